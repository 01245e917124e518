// Shared by the kernels that attend over the 4-bit cache.
//
//   s_rj = scale * q_r . k_j,  k_j = lo_j + step_j c_j  =>  s_rj = scale * (step_j (q_r . c_j) + lo_j sum(q_r))
//   o_r  = sum_j p_rj v_j / sum_j p_rj                  =   (sum_j (p_rj step_j) c_j + sum_j p_rj lo_j) / sum_j p_rj
//
// so the matrix products run on the 4-bit codes themselves and a token's two parameters enter the scores and
// the probabilities, not the elements: nothing of K or V is rounded. A code needs one AND to become an
// operand: in the low bits of a half it is the subnormal c * 2^-24, four bits higher c * 2^-20, both exact,
// and the powers of two go into q and the result. (The sum of products is another matter: the values' codes of the
// kernel for few rows stand higher, see there.)
// q is multiplied by the power of two that puts its row's largest element into [2^13, 2^14), in the kernel for many rows
// into [2^15, 2^16): fp16 then holds bf16's eight bits exactly down to 2^-28 of the largest element (and fp16's eleven to
// 2^-25).
// The weights w = p * step of the second product are rounded to fp16 (2^-11). p is 2^(s - m) with an m of the row's own
// that follows s + log2(step) over the tokens the row sees (exponents rounded up, a lag of 2^8 allowed): w stays below
// 2^15, and the largest is 2^6 or more (2^-2 in the kernel for many rows, which takes a tile's largest score and largest
// step together where its steps are within 2^8), so that what is lost of a subnormal weight is 2^-23 of the largest at
// most. Nothing that a row does not see, and nothing that weighs nothing in it, enters m. (Divided by the largest step of
// all tokens in the row's tiles, weights lost the bits by which a hidden value was larger: of 300 tokens the error grew
// from 1.8e-3 to 2.1e-3 beside one 2^16 times larger, to 1.4e-2 at 2^20.)
// With w the rounded weight the result is formed as sum w c - 7.5 sum w + sum p (lo + 7.5 step) (the kernel for many rows:
// 8): the rounding then acts on c - 7.5, at most half as large as c. With sum w c and lo the error of an fp16 result was
// 2.9 times its own rounding; so it is 1.45 to 1.57 times (512 rows over 2048 tokens, 256 and 64 elements; a bf16
// result's is its rounding, 1.01 times), which the kernel for few rows brings to 1.00 with a second product. The one for
// many rows leaves it: its softmax warps, which bound it, would issue a third more.
#pragma once

#include "kvcache.cuh"

namespace b200lut {

// Sums of a row's elements are held in units of 2^9: finite for every row, and exact for the smallest elements too.
constexpr float kSumUnit = 1.f / 512.f;

struct AttendParams {
  const uint16_t* q;
  const uint16_t* gate;        // or null
  uint16_t* out;
  long long q_token, q_head, gate_token, gate_head, out_token, out_head;    // strides in elements
  CacheView c;
  const int* table;
  const int* kv_len;
  const int* row_start;        // or null: one row per request
  long long table_ld;
  int T, B, Hq, G, width, window, sinks;     // T * G < 2^31
  uint32_t g_mul;              // x / G = umulhi(x, g_mul) >> g_shift for x < 2^31 (G = 1: x)
  int g_shift;
  float scale;                 // scale * log2(e)
  // a request of at most so many rows (times query heads per key/value head) is the single-row kernel's, the
  // others are the tile kernel's; INT_MAX: no tile kernel runs
  int rows_limit;
  long long wait_cycles;
  // workspace: per block, what it left to be joined
  int4* meta;
  float2* part_ml;
  float* part_o;
};

// Row r of a request's head is its token r / G and the head's query head r % G.
__device__ __forceinline__ int token_of(const AttendParams& p, int r) {
  return p.G == 1 ? r : int(__umulhi(uint32_t(r), p.g_mul) >> p.g_shift);
}

// The requests' rows and lengths as the kernels read them (device data: clamped, never trusted).
struct Request {
  int row0, rows, len;         // first row, rows, cached tokens with them
};
__device__ __forceinline__ Request request_of(const AttendParams& p, int b) {
  Request r;
  r.row0 = p.row_start ? min(max(0, p.row_start[b]), p.T) : b;
  r.rows = p.row_start ? max(0, min(p.row_start[b + 1], p.T) - r.row0) : 1;
  const long long room = (long long)p.width << p.c.page_log2;
  const int len = max(0, p.kv_len[b]);
  r.len = int(min((long long)len, room));
  return r;
}

// What the join has to know of an item that a block began: the last block of it, the row of q of the item's first row's
// token, and packed: rows - 1, how far the first row is into its token's query heads, key/value head.
__device__ __forceinline__ int4 joined_item(const AttendParams& p, int last, const Request& rq, int h, int r0, int n_rows) {
  const int tok = token_of(p, r0);
  return make_int4(last, rq.row0 + tok, 0, (n_rows - 1) | ((r0 - tok * p.G) << 7) | (h << 13));
}

// Tiles of kTile tokens that rows at positions [first, last] of a request see: ids 0 .. sink_tiles - 1, then from
// main0 on. At least one, so that a row that sees nothing is written.
template <int kTile>
struct Span {
  int sink_tiles, main0, tiles;
  __device__ Span() {}
  __device__ __forceinline__ Span(int first, int last, int len, int window, int sinks) {
    const int hi = min(len, last + 1);                       // tokens below hi
    const int lo = window && first >= window ? first - window + 1 : 0;      // rows before the sequence: no difference wraps
    const int s = min(min(sinks, lo), max(hi, 0));
    sink_tiles = tiles_of(s);
    main0 = max(lo / kTile, sink_tiles);
    const int main1 = tiles_of(max(hi, 0));
    tiles = max(1, sink_tiles + max(0, main1 - main0));
  }
  // up to 2^31 - 1 tokens: the sum n + kTile - 1 would wrap
  static __device__ __forceinline__ int tiles_of(int n) { return int((unsigned(n) + (kTile - 1)) / kTile); }
  __device__ __forceinline__ int id(int i) const { return i < sink_tiles ? i : main0 + i - sink_tiles; }
};

__device__ __forceinline__ bool token_seen(int j, int pos, int len, int window, int sinks) {
  return j <= pos && j < len && (window == 0 || pos - j < window || j < sinks);
}

template <typename T>
__device__ __forceinline__ float gated(float o, const AttendParams& p, long long token, int head, int d) {
  if (!p.gate) return o;
  const float g = DType<T>::to_float(p.gate[token * p.gate_token + (long long)head * p.gate_head + d]);
  return o / (1.f + __expf(-g));
}

// A token's size: its step, or 2^-20 of its middle where that is larger (a row of equal elements has no step), or 2^-94;
// so p * step and p * mid both keep their range. What it adds to a score in m: the exponent of the next power of two, less
// the 7 that leave weights room up to 2^7, 2^15 with the lag.
// m of two parts of a row may differ by some 200 for the tokens' sizes alone: a sum of p takes the factor between them in
// two halves, since the sum may be as large as the factor is small.
constexpr float kMinStep = 5.04870979e-29f;      // 2^-94
__device__ __forceinline__ float token_size(float step, float mid) { return fmaxf(step, fmaxf(fabsf(mid) * 9.5367432e-7f, kMinStep)); }
__device__ __forceinline__ int exponent_above(float size) { return int((__float_as_uint(size) + 0x007FFFFFu) >> 23) - 127; }
__device__ __forceinline__ float size_in_m(float size) { return float(exponent_above(size) - 7); }

// The tile kernel over `blocks` blocks (its joins are launched with those of the row kernel).
int attend_tiles(const AttendParams& p, int dtype, int blocks, cudaStream_t stream);

}  // namespace b200lut
