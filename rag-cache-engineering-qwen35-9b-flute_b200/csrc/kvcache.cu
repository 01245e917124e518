// The paged 4-bit key/value cache: the step plan (row starts, positions, page assignment and slots from the
// requests' lengths, on the device), rows written and rows read back. Layout: kvcache.cuh.
#include <type_traits>

#include "kvcache.cuh"
#include "packed.cuh"

namespace b200lut {
namespace {

__device__ int g_kv_status = 0;
constexpr int kBadSlot = 0x6100;

// ---- step plan ------------------------------------------------------------------------------------------
// One launch: every block scans all requests (two sums: new tokens and pages wanted; a scan over 1024
// requests is one block-wide scan), then fills its share of the tokens. A token's page is either an entry of
// the request's row or, past the pages it has, the next of the free list, so no block waits for another; the
// entry of a fresh page is written by the thread of that page's first token.
struct PlanParams {
  const int *cached, *fresh;
  int* table;
  const int *free_pages, *taken;
  int *row_start, *kv_len, *positions, *slots, *taken_out;
  uint8_t* served;
  int B, width, free_count, page_log2, max_tokens;
};

constexpr int kUnserved = INT32_MIN;

__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int sm[];
  int* end = sm;                 // [B] tokens up to and with request b, clamped to 2^31 - 1
  int* base = sm + p.B;          // [B] free-list index of page j of request b, less j; kUnserved
  __shared__ long long warp_tokens[32], warp_pages[32];
  __shared__ int taken_max;
  const int n = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = 1 << p.page_log2;
  const int taken = max(0, *p.taken);
  if (tid == 0) taken_max = taken;
  long long carry_tokens = 0, carry_pages = taken;
  for (int b0 = 0; b0 < p.B; b0 += n) {
    const int b = b0 + tid;
    long long cached = 0, fresh = 0;
    if (b < p.B) cached = max(0, p.cached[b]), fresh = max(0, p.fresh[b]);
    // tokens first: whether a request fits depends on where its rows end
    long long tok = fresh;
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, tok, o);
      if (lane >= o) tok += v;
    }
    if (lane == 31) warp_tokens[warp] = tok;
    __syncthreads();
    long long before = carry_tokens;
    for (int w = 0; w < n / 32; ++w) {
      if (w < warp) before += warp_tokens[w];
      carry_tokens += warp_tokens[w];
    }
    tok += before;
    const long long have = (cached + P - 1) >> p.page_log2, want = (cached + fresh + P - 1) >> p.page_log2;
    // positions and lengths are 32-bit: past them a page index would be negative
    const bool fits = b < p.B && want <= p.width && tok <= p.max_tokens && cached + fresh <= INT32_MAX;
    const long long need = fits ? want - have : 0;
    long long pg = need;
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, pg, o);
      if (lane >= o) pg += v;
    }
    if (lane == 31) warp_pages[warp] = pg;
    __syncthreads();
    long long used = carry_pages;
    for (int w = 0; w < n / 32; ++w) {
      if (w < warp) used += warp_pages[w];
      carry_pages += warp_pages[w];
    }
    pg += used;
    if (b < p.B) {
      const bool served = fits && (need == 0 || pg <= p.free_count);
      end[b] = int(min(tok, (long long)INT32_MAX));
      base[b] = served ? int(pg - need - have) : kUnserved;
      if (served && need > 0) atomicMax(&taken_max, int(pg));
      if (blockIdx.x == 0) {
        p.row_start[b] = int(min(tok - fresh, (long long)p.max_tokens));
        if (b == p.B - 1) p.row_start[p.B] = int(min(tok, (long long)p.max_tokens));
        p.kv_len[b] = int(served ? cached + fresh : cached);
        p.served[b] = served ? 1 : 0;
      }
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) *p.taken_out = taken_max;
  const int total = end[p.B - 1];
  for (int t = blockIdx.x * n + tid; t < p.max_tokens; t += gridDim.x * n) {
    int pos = 0, slot = -1;
    if (t < total) {
      int lo = 0, hi = p.B - 1;                  // first request that ends behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int b = lo, cached = max(0, p.cached[b]);
      // of a request that is not the first in a clamped sum, the start is exact whenever t lies in it
      const int start = b ? end[b - 1] : 0;
      pos = int(min((long long)cached + (t - start), (long long)INT32_MAX));
      if (base[b] != kUnserved) {
        const int j = pos >> p.page_log2;
        int* entry = p.table + (long long)b * p.width + j;
        int page;
        if (j >= int(((long long)cached + P - 1) >> p.page_log2)) {
          page = p.free_pages[base[b] + j];
          if ((pos & (P - 1)) == 0) *entry = page;
        } else {
          page = *entry;
        }
        // a page that is none: a slot that a write reports
        if (page >= 0) slot = page > (INT32_MAX >> p.page_log2) ? INT32_MAX : (page << p.page_log2) + (pos & (P - 1));
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// ---- rows in ------------------------------------------------------------------------------------------
// A row is D/8 lanes of eight elements: two shuffle reductions give lo and hi, then each lane writes the one
// 32-bit word of codes its elements make. A warp takes the rows of U consecutive tokens, all loaded before the first is
// worked on; four tokens whose slots are neighbours (a prompt's) make 16-byte stores of the values. Rows are read once,
// codes written once, but the bound is issue, not memory: 16384 tokens of 4 heads of 256 take 31 us (reading them back
// 17), where their 84 MB would take 13. So elements stay in 16-bit pairs until the codes are made: the extremes are one
// packed maximum over (x, -x), which keeps NaN, one shuffle moves both, and everything behind them is two elements an
// instruction (47 us with one element an instruction, 33 with the head's width as an argument, 27 without the decisions in
// 64 bits that borders need).
constexpr int kRowWarps = 4;
constexpr float kRangeLimit = 1.329227996e36f;     // 2^120: 15 times a range below it is finite

// rint(a / w), half to even, of both halves, 0 <= a <= 15 w, with inv = 1 / w rounded; the second half's code at bit 4.
// The quotient is the correctly rounded one (Markstein: the residual a - q w of a quotient that is off by an ulp, times
// the rounded reciprocal, added to it), so codes on a border, frequent with eight-bit significands, are decided as the
// definition does. Adding 1.5 * 2^23 then rounds to an integer and leaves it in the low bits. `far`: the largest
// distance of a quotient from its code.
template <bool kFar>
__device__ __forceinline__ uint32_t two_codes(float2 a, float2 minus_w, float2 inv, float* far) {
  const float2 magic = make_float2(12582912.f, 12582912.f);
  float2 q = mul2(a, inv);
  q = fma2(fma2(q, minus_w, a), inv, q);
  const float2 m = add2(q, magic);
  if constexpr (kFar) {
    const float2 n = add2(m, make_float2(-12582912.f, -12582912.f));
    const float2 d = add2(q, make_float2(-n.x, -n.y));
    *far = fmaxf(*far, fmaxf(fabsf(d.x), fabsf(d.y)));
  }
  return (__float_as_uint(m.x) & 15u) | ((__float_as_uint(m.y) & 15u) << 4);
}

template <typename T, int D, int U>
__global__ void __launch_bounds__(kRowWarps * 32) kv_write_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                                  long long kt, long long kh, long long vt, long long vh,
                                                                  const int* __restrict__ slots, int tokens, CacheView c) {
  constexpr int lanes = D / 8, per = 32 / lanes;
  const int lane = threadIdx.x & 31, at = lane % lanes;
  const unsigned row = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * per + lane / lanes;
  const unsigned half = (unsigned(tokens) + U - 1) / U * unsigned(c.heads);      // 2 half < 2^31
  const bool in = row < 2 * half, value = row >= half;
  const unsigned r = in ? (value ? row - half : row) : 0, group = r / unsigned(c.heads);
  const int h = int(r - group * c.heads), t0 = int(group) * U;
  int slot[U];
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u;
    slot[u] = -1;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (in && t < tokens) {
      slot[u] = slots[t];
      const uint16_t* x = value ? v + t * vt + h * vh : k + t * kt + h * kh;
      raw[u] = __ldg(reinterpret_cast<const uint4*>(x) + at);
    }
  }
  uint32_t word[U], pair[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    // (hi, -lo) as one 16-bit pair: a NaN stays one
    uint32_t top = max2_nan(max2_nan(w[0], w[1], T()), max2_nan(w[2], w[3], T()), T());
    uint32_t low = max2_nan(max2_nan(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u, T()),
                            max2_nan(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u, T()), T());
    uint32_t ends = max2_nan(__byte_perm(top, low, 0x5410), __byte_perm(top, low, 0x7632), T());
#pragma unroll
    for (int o = lanes >> 1; o; o >>= 1) ends = max2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, o), T());
    const float2 hl = unpack2(ends, T());
    const float lo = -hl.y, range = hl.x - lo;
    const bool finite = range < kRangeLimit;               // false for NaN too
    word[u] = 0;
    if (finite && range > 0.f) {
      // scaled by a power of two that keeps 1 / range and the products normal
      const float up = range < 1e-30f ? 1.329227996e36f : 1.f, width = range * up, inv = 1.f / width;
      const float by = 15.f * up;                          // products with it are exact
      const float2 inv2 = make_float2(inv, inv), minus = make_float2(-width, -width), scale = make_float2(by, by);
      const float2 low = make_float2(-lo * by, -lo * by);
      // a has more than fp32's 24 bits where x and lo lie more than 2^12 apart (fp16, of longer significands: 2^8). What
      // then comes near to a border is decided in 64 bits: in fp16 any such quotient (one warp in some hundred); in bf16
      // the rows where it can happen, those with an end far below the other and those whose zero lies at a border.
      constexpr bool kFar = std::is_same<T, __half>::value;
      float far = 0.f;
      if constexpr (!kFar) {
        const float ends_lo = fminf(fabsf(lo), fabsf(hl.x)), zero = low.x * inv;
        if (ends_lo < 4.8828125e-4f * fmaxf(fabsf(lo), fabsf(hl.x)) ? ends_lo != 0.f : fabsf(zero - rintf(zero)) > 0.496f) far = 1.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        word[u] |= two_codes<kFar>(fma2(unpack2(w[e], T()), scale, low), minus, inv2, &far) << (8 * e);
      if (far > 0.49999f) {
        word[u] = 0;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint32_t pair_of = e < 2 ? w[0] : e < 4 ? w[1] : e < 6 ? w[2] : w[3];
          const float2 x = unpack2(pair_of, T());
          const double q = 15.0 * (double(e & 1 ? x.y : x.x) - double(lo)) / (double(hl.x) - double(lo));
          word[u] |= uint32_t(__double2int_rn(q)) << (4 * e);
        }
      }
    }
    pair[u] = finite ? __byte_perm(ends ^ 0x80000000u, 0, 0x1032) : 0x7FFF7FFFu;       // lo in the low half
  }
  const int limit = c.n_pages << c.page_log2;
  if constexpr (U == 4) {
    // four neighbours at a boundary of four (they share a page and a 16-token block)
    if (value && slot[0] >= 0 && slot[0] < limit && (slot[0] & 3) == 0 && slot[1] == slot[0] + 1 && slot[2] == slot[0] + 2 &&
        slot[3] == slot[0] + 3) {
      const int page = slot[0] >> c.page_log2, offset = slot[0] & ((1 << c.page_log2) - 1);
      *reinterpret_cast<uint4*>(c.v + cache_codes_at(page, h, c.heads, c.page_log2, D) + value_word_at(offset, at, D)) =
          make_uint4(word[0], word[1], word[2], word[3]);
      if (at == 0)
        *reinterpret_cast<uint4*>(c.v_pair + cache_pair_at(page, h, c.heads, c.page_log2, offset)) =
            make_uint4(pair[0], pair[1], pair[2], pair[3]);
      return;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] < 0) continue;
    if (slot[u] >= limit) {
      if (at == 0) atomicExch(&g_kv_status, kBadSlot);
      continue;
    }
    const int page = slot[u] >> c.page_log2, offset = slot[u] & ((1 << c.page_log2) - 1);
    uint8_t* codes = (value ? c.v : c.k) + cache_codes_at(page, h, c.heads, c.page_log2, D);
    *reinterpret_cast<uint32_t*>(codes + (value ? value_word_at(offset, at, D) : key_word_at(offset, at, D))) = word[u];
    if (at == 0) (value ? c.v_pair : c.k_pair)[cache_pair_at(page, h, c.heads, c.page_log2, offset)] = pair[u];
  }
}

// ---- rows out -----------------------------------------------------------------------------------------
// The same shape: U tokens of a row's lane, all words under way before the first is unpacked.
template <typename T, int D, int U>
__global__ void __launch_bounds__(kRowWarps * 32) kv_read_kernel(uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                                 const int* __restrict__ slots, int tokens, CacheView c) {
  constexpr int lanes = D / 8, per = 32 / lanes;
  const int lane = threadIdx.x & 31, at = lane % lanes;
  const unsigned row = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * per + lane / lanes;
  const unsigned half = (unsigned(tokens) + U - 1) / U * unsigned(c.heads);      // 2 half < 2^31
  if (row >= 2 * half) return;
  const bool value = row >= half;
  const unsigned r = value ? row - half : row, group = r / unsigned(c.heads);
  const int h = int(r - group * c.heads), t0 = int(group) * U;
  const int limit = c.n_pages << c.page_log2;
  uint32_t word[U], pair[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    word[u] = pair[u] = 0;
    const int slot = t0 + u < tokens ? slots[t0 + u] : -1;
    if (slot >= limit) {
      if (at == 0) atomicExch(&g_kv_status, kBadSlot);
    } else if (slot >= 0) {
      const int page = slot >> c.page_log2, offset = slot & ((1 << c.page_log2) - 1);
      const uint8_t* codes = (value ? c.v : c.k) + cache_codes_at(page, h, c.heads, c.page_log2, D);
      word[u] = *reinterpret_cast<const uint32_t*>(codes + (value ? value_word_at(offset, at, D) : key_word_at(offset, at, D)));
      pair[u] = (value ? c.v_pair : c.k_pair)[cache_pair_at(page, h, c.heads, c.page_log2, offset)];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (t0 + u >= tokens) break;
    const float2 ls = lo_step<T>(pair[u]), lo2 = make_float2(ls.x, ls.x), step2 = make_float2(ls.y, ls.y);
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {        // 2^23 + code, less 2^23
      const float2 n = make_float2(__uint_as_float(((word[u] >> (8 * e)) & 15u) | 0x4B000000u),
                                   __uint_as_float(((word[u] >> (8 * e + 4)) & 15u) | 0x4B000000u));
      out[e] = pack2(fma2(add2(n, make_float2(-8388608.f, -8388608.f)), step2, lo2), T());
    }
    reinterpret_cast<uint4*>((value ? v : k) + ((long long)(t0 + u) * c.heads + h) * D)[at] = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// Tokens a warp takes: one while a wave of warps (32 an SM) holds every row, four beyond.
inline int tokens_per_warp(long long rows, int D) { return rows * D <= 256LL * 148 * 32 ? 1 : 4; }

}  // namespace

int kv_status_take() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kv_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_kv_status, &zero, sizeof(int));
  return v;
}

int check_cache(const b200lut_kv_cache* c, const char* who, CacheView* v) {
  B200LUT_REQUIRE(c && c->k_codes && c->v_codes && c->k_pairs && c->v_pairs, B200LUT_ERR_INVALID, "%s: null cache", who);
  B200LUT_REQUIRE(c->dtype == B200LUT_BF16 || c->dtype == B200LUT_F16, B200LUT_ERR_INVALID,
                  "%s: dtype must be B200LUT_BF16 or B200LUT_F16", who);
  B200LUT_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, B200LUT_ERR_UNSUPPORTED,
                  "%s: head_dim must be 64, 128 or 256 (got %d)", who, c->head_dim);
  B200LUT_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
                  B200LUT_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64, 128 or 256 (got %d)", who, c->page_size);
  B200LUT_REQUIRE(c->n_kv_heads >= 1 && c->n_kv_heads <= 4096 && c->n_pages >= 1 &&
                      (long long)c->n_pages * c->page_size <= 0x7fffffffLL,
                  B200LUT_ERR_INVALID, "%s: 1 to 4096 heads and fewer than 2^31 slots wanted", who);
  B200LUT_REQUIRE(aligned16(c->k_codes) && aligned16(c->v_codes) && aligned16(c->k_pairs) && aligned16(c->v_pairs),
                  B200LUT_ERR_ALIGN, "%s: cache buffers must be 16-byte aligned", who);
  v->k = static_cast<uint8_t*>(c->k_codes), v->v = static_cast<uint8_t*>(c->v_codes);
  v->k_pair = static_cast<uint32_t*>(c->k_pairs), v->v_pair = static_cast<uint32_t*>(c->v_pairs);
  v->n_pages = c->n_pages, v->heads = c->n_kv_heads, v->D = c->head_dim;
  v->page_log2 = 31 - __builtin_clz(unsigned(c->page_size));
  return B200LUT_OK;
}

}  // namespace b200lut

using namespace b200lut;

extern "C" int b200lut_kv_plan(const b200lut_kv_plan_args* a, void* stream) {
  B200LUT_REQUIRE(a && a->cached && a->fresh && a->block_table && a->free_pages && a->taken && a->row_start && a->kv_len &&
                      a->positions && a->slots && a->taken_out && a->served,
                  B200LUT_ERR_INVALID, "kv_plan: null argument");
  B200LUT_REQUIRE(a->B >= 1 && a->B <= 8192, B200LUT_ERR_UNSUPPORTED, "kv_plan: 1 to 8192 requests (got %d)", a->B);
  B200LUT_REQUIRE(a->width >= 1 && a->free_count >= 0 && a->max_tokens >= 1, B200LUT_ERR_INVALID,
                  "kv_plan: width and max_tokens must be positive, free_count not negative");
  B200LUT_REQUIRE(a->page_size >= 16 && a->page_size <= 256 && (a->page_size & (a->page_size - 1)) == 0,
                  B200LUT_ERR_UNSUPPORTED, "kv_plan: page_size must be 16, 32, 64, 128 or 256 (got %d)", a->page_size);
  PlanParams p;
  p.cached = a->cached, p.fresh = a->fresh, p.table = a->block_table, p.free_pages = a->free_pages, p.taken = a->taken;
  p.row_start = a->row_start, p.kv_len = a->kv_len, p.positions = a->positions, p.slots = a->slots;
  p.taken_out = a->taken_out, p.served = a->served;
  p.B = a->B, p.width = a->width, p.free_count = a->free_count, p.max_tokens = a->max_tokens;
  p.page_log2 = 31 - __builtin_clz(unsigned(a->page_size));
  const int n = a->B <= 128 ? 128 : a->B <= 512 ? 512 : 1024;
  long long grid = ((long long)a->max_tokens + n - 1) / n;
  if (grid > 148) grid = 148;
  const size_t smem = size_t(a->B) * 8;
  if (smem > 40 * 1024)
    B200LUT_CUDA_OK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8192 * 8));
  plan_kernel<<<unsigned(grid), n, smem, cudaStream_t(stream)>>>(p);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}

extern "C" int b200lut_kv_write(const b200lut_kv_cache* cache, const void* k, const void* v, int64_t k_token_stride,
                                int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                const int32_t* slots, int tokens, void* stream) {
  CacheView c;
  const int rc = check_cache(cache, "kv_write", &c);
  if (rc != B200LUT_OK) return rc;
  B200LUT_REQUIRE(tokens >= 0 && (tokens == 0 || (k && v && slots)), B200LUT_ERR_INVALID, "kv_write: null argument");
  B200LUT_REQUIRE(aligned16(k) && aligned16(v) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                      v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                  B200LUT_ERR_ALIGN, "kv_write: rows must be 16-byte aligned (pointers and strides)");
  if (tokens == 0) return B200LUT_OK;
  const int U = tokens_per_warp(2LL * tokens * c.heads, c.D);
  const long long rows = 2LL * ((tokens + U - 1LL) / U) * c.heads, per = (256 / c.D) * kRowWarps, grid = (rows + per - 1) / per;
  B200LUT_REQUIRE(rows <= 0x7fffff00LL && tokens <= 0x7fffff00, B200LUT_ERR_UNSUPPORTED, "kv_write: too many rows");
  const auto* kk = static_cast<const uint16_t*>(k);
  const auto* vv = static_cast<const uint16_t*>(v);
  const bool bf = cache->dtype == B200LUT_BF16;
  const auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return U == 1 ? (bf ? kv_write_kernel<__nv_bfloat16, D, 1> : kv_write_kernel<__half, D, 1>)
                  : (bf ? kv_write_kernel<__nv_bfloat16, D, 4> : kv_write_kernel<__half, D, 4>);
  };
  auto* kernel = c.D == 64 ? pick(std::integral_constant<int, 64>()) : c.D == 128 ? pick(std::integral_constant<int, 128>())
                                                                                 : pick(std::integral_constant<int, 256>());
  kernel<<<unsigned(grid), kRowWarps * 32, 0, cudaStream_t(stream)>>>(kk, vv, k_token_stride, k_head_stride, v_token_stride,
                                                                      v_head_stride, slots, tokens, c);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}

extern "C" int b200lut_kv_read(const b200lut_kv_cache* cache, void* k, void* v, const int32_t* slots, int tokens,
                               void* stream) {
  CacheView c;
  const int rc = check_cache(cache, "kv_read", &c);
  if (rc != B200LUT_OK) return rc;
  B200LUT_REQUIRE(tokens >= 0 && (tokens == 0 || (k && v && slots)), B200LUT_ERR_INVALID, "kv_read: null argument");
  B200LUT_REQUIRE(aligned16(k) && aligned16(v), B200LUT_ERR_ALIGN, "kv_read: outputs must be 16-byte aligned");
  if (tokens == 0) return B200LUT_OK;
  const int U = tokens_per_warp(2LL * tokens * c.heads, c.D);
  const long long rows = 2LL * ((tokens + U - 1LL) / U) * c.heads, per = (256 / c.D) * kRowWarps, grid = (rows + per - 1) / per;
  B200LUT_REQUIRE(rows <= 0x7fffff00LL && tokens <= 0x7fffff00, B200LUT_ERR_UNSUPPORTED, "kv_read: too many rows");
  auto* kk = static_cast<uint16_t*>(k);
  auto* vv = static_cast<uint16_t*>(v);
  const bool bf = cache->dtype == B200LUT_BF16;
  const auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return U == 1 ? (bf ? kv_read_kernel<__nv_bfloat16, D, 1> : kv_read_kernel<__half, D, 1>)
                  : (bf ? kv_read_kernel<__nv_bfloat16, D, 4> : kv_read_kernel<__half, D, 4>);
  };
  auto* kernel = c.D == 64 ? pick(std::integral_constant<int, 64>()) : c.D == 128 ? pick(std::integral_constant<int, 128>())
                                                                                 : pick(std::integral_constant<int, 256>());
  kernel<<<unsigned(grid), kRowWarps * 32, 0, cudaStream_t(stream)>>>(kk, vv, slots, tokens, c);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}
