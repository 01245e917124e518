// Attention over the 4-bit cache for many rows per request (prompts, chunks of prompts): tcgen05 on codes.
//
// A work item is 128 rows (query heads of one key/value head, times new tokens) of one request; its visible
// tokens are cut into tiles of 128. All items' tiles form one line that is dealt to the blocks (one per SM) in
// equal contiguous shares; items that span blocks are joined by a second kernel in the order of the blocks.
// Per tile, in the roles of one block:
//   warp 14     parameters: pages, and what the tokens' pairs say (one tile ahead of everybody else).
//   warps 12-13 keys: codes from global memory (fetched one tile ahead) into fp16 operands in shared memory, 128-byte
//               swizzle, [token, dim] rows.
//   warps 8-11  values: transposed, [dim, token] rows. A 16-byte piece holds four tokens' words side by side, two byte
//               permutes make pairs of tokens. The words are rotated by the lane's group first, so that the
//               eight rows a store hits differ in their swizzle.
//   warp 15     one thread issues S = Q K^T (128 x 128, fp32 in tensor memory, two buffers) and O += P V (128 x D).
//   warps 0-7   softmax, two threads a row (64 tokens each): scores from tensor memory, the token's two parameters
//               applied as packed pairs, P back into the place of S as fp16 (the A operand of the second product).
//               The running maximum may lag by 2^8 before O is rescaled, which then waits for the products in flight.
// Tensor memory: O in columns 0 .. D - 1, S in 256 .. 383 and 384 .. 511.
#include "attend.cuh"
#include "tc05.cuh"

namespace b200lut {
namespace {

__device__ int g_tiles_status = 0;
constexpr int kRows = 128, kTile = 128;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kValueWarp = 8, kKeyWarp = 12, kParamWarp = 14, kProductWarp = 15;
constexpr int kParamStages = 4;
constexpr float kLazy = 8.f;
constexpr float kMinStep = 7.888609e-31f;   // 2^-100
constexpr int kBadPage = 0x6200;

template <int D>
struct Shape {
  static constexpr int kStages = D == 256 ? 1 : 2;
  static constexpr int kOperand = 256 * D;                       // bytes of 128 x D halves
  static constexpr int kQ = 0, kK = kOperand, kV = kK + kStages * kOperand;
  static constexpr int kParam = kV + kStages * kOperand;         // [stage][64 token pairs] of a, a, lo, lo and s, s, mid, mid
  static constexpr int kParamBytes = 2 * 64 * 16;
  static constexpr int kEnd = kParam + kParamStages * kParamBytes;
  static constexpr int kSmem = kEnd + 1024;                      // the base is rounded up to 1024
};

struct TileInfo {
  float sig;                   // power of two >= the largest step so far
  int whole;                   // every row sees every token
  uint32_t valid[4];           // tokens that some row may see
  int page[8];                 // of each 16 tokens; -1: none
};

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float pow2_above(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x007FFFFFu) & 0x7F800000u);
}
__device__ __forceinline__ uint32_t half2_of(float2 a) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(a.y), "f"(a.x));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// D[d] (+)= A[desc a] B[desc b], one K = 16 step; one thread issues.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"(accumulate), "r"(0u)
      : "memory");
}

__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// ---- the line of tiles ---------------------------------------------------------------------------------------
__device__ __forceinline__ Request tiles_request(const AttendParams& p, int b) {
  Request r = request_of(p, b);
  if ((long long)r.rows * p.G <= p.rows_limit) r.rows = 0;       // the other kernel's
  return r;
}
__device__ __forceinline__ Span<kTile> span_of(const AttendParams& p, const Request& r, long long r0) {
  const long long rows = (long long)r.rows * p.G;
  const int base = r.len - r.rows;
  const long long last = min(r0 + kRows, rows) - 1;
  return Span<kTile>(base + int(r0 / p.G), base + int(last / p.G), r.len, p.window, p.sinks);
}
// Tiles of one head of request b, summed over its row tiles by a whole warp (all lanes get the sum).
__device__ __forceinline__ long long head_tiles(const AttendParams& p, const Request& r, int lane) {
  const long long n = ((long long)r.rows * p.G + kRows - 1) / kRows;
  long long sum = 0;
  for (long long i = lane; i < n; i += 32) sum += span_of(p, r, i * kRows).tiles;
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// A part of an item: tiles [i0, i1) of row tile rt of head h of request b.
struct Work {
  int b, h;
  long long rt;
  int i0, i1, tiles;
  Request rq;
  long long item_at;           // tiles of the line before the item
};

// What the roles need of it.
struct Item {
  Span<kTile> span;
  long long r0;
  int n_rows, base, first_pos, last_pos;
  uint32_t n0;                 // tiles of this block before the item's
  int count;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) attend_tiles_kernel(const __grid_constant__ AttendParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw_sm[];
  __shared__ __align__(8) uint64_t bars[32];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  __shared__ float2 row_k[kRows];              // factor of the scores, sum of the scaled row
  __shared__ TileInfo info[kParamStages];
  __shared__ float half_top[2][2][kRows];      // [tile & 1][half][row]
  __shared__ float2 half_sum[kRows];
  __shared__ long long scan[kWarps];
  __shared__ long long first_at;
  __shared__ int first_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sm = (tc::smem_addr(raw_sm) + 1023u) & ~1023u;
  const uint32_t base_off = sm - tc::smem_addr(raw_sm);
  volatile int* abort_flag = &abort_word;
  const uint32_t bar0 = tc::smem_addr(bars);
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  // keys are handed over in blocks of 64 elements, values in blocks of 64 tokens: [stage][block]
  constexpr int kKB = D / 64, kKBars = S::kStages * kKB, kVBars = S::kStages * 2;
  constexpr int kKFull = 0, kKEmpty = 4, kVFull = 8, kVEmpty = 12, kSFull = 16, kPFull = 18, kPvDone = 20, kPrmFull = 22,
                kPrmEmpty = 26;
  static_assert(kKBars <= 4 && kVBars <= 4, "barriers");

  // ---- this block's share
  if (tid == 0) {
    p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    abort_word = 0;
    first_b = p.B;
  }
  const int per = (p.B + kWarps - 1) / (kWarps);
  long long mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = warp * per + i;
    if (b < p.B) mine += head_tiles(p, tiles_request(p, b), lane) * p.c.heads;
  }
  if (lane == 0) scan[warp] = mine;
  __syncthreads();
  long long total = 0, before = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const long long share = max(1LL, (total + gridDim.x - 1) / gridDim.x);
  const long long begin = share * blockIdx.x, stop = min(total, begin + share);
  if (begin >= stop) return;
  if (begin >= before && begin < before + mine) {
    long long at = before;
    for (int i = 0; i < per; ++i) {
      const int b = warp * per + i;
      if (b >= p.B) break;
      const long long n = head_tiles(p, tiles_request(p, b), lane) * p.c.heads;
      if (begin < at + n) {
        if (lane == 0) first_b = b, first_at = at;
        break;
      }
      at += n;
    }
  }
  if (warp == kProductWarp) tc::tmem_alloc(tc::smem_addr(&tmem_base), 512);
  if (tid == 0) {
    for (int i = 0; i < kKBars; ++i) tc::mbar_init(bar(kKFull + i), 2), tc::mbar_init(bar(kKEmpty + i), 1);
    for (int i = 0; i < kVBars; ++i) tc::mbar_init(bar(kVFull + i), 2), tc::mbar_init(bar(kVEmpty + i), 1);
    for (int i = 0; i < 2; ++i)
      tc::mbar_init(bar(kSFull + i), 1), tc::mbar_init(bar(kPFull + i), 8), tc::mbar_init(bar(kPvDone + i), 1);
    for (int i = 0; i < kParamStages; ++i) tc::mbar_init(bar(kPrmFull + i), 1), tc::mbar_init(bar(kPrmEmpty + i), 14);
    tc::mbar_init_fence();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  auto wait = [&](int i, uint32_t parity, int why) {
    tc::mbar_wait(bar(i), parity, abort_flag, &g_tiles_status, why, p.wait_cycles);
  };

  // A wait names a phase by its parity alone: whoever waits must know that the phase before is complete and that
  // the one after cannot be yet. Product P V of tile m reports to barrier m & 1: tile m - 2 is through when S of m is
  // there, tile m + 2 waits for P of m.
  auto wait_pv = [&](uint32_t m) { wait(kPvDone + int(m & 1), (m >> 1) & 1u, tc::kStatusWaitDone); };

  // the first item (every warp finds it by itself)
  Work w;
  w.b = first_b;
  {
    w.rq = tiles_request(p, w.b);
    const long long per_head = head_tiles(p, w.rq, lane);
    long long off = begin - first_at;
    w.h = int(off / per_head);
    off -= w.h * per_head;
    const long long n = ((long long)w.rq.rows * p.G + kRows - 1) / kRows;
    w.rt = 0;
    for (long long c0 = 0; c0 < n; c0 += 32) {
      const long long tiles = c0 + lane < n ? span_of(p, w.rq, (c0 + lane) * kRows).tiles : 0;
      long long inc = tiles;
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, off < inc);
      if (hit) {
        const int l = __ffs(int(hit)) - 1;
        w.rt = c0 + l;
        off -= __shfl_sync(0xffffffffu, inc - tiles, l);
        break;
      }
      off -= __shfl_sync(0xffffffffu, inc, 31);
    }
    w.item_at = begin - off;
  }

  uint32_t n = 0;                              // tiles of this block so far
  // Every role walks the block's items: the rows' operand is made by all warps, then `body` does the role's
  // part of the item's tiles.
  auto items = [&](auto&& body) {
    long long cur = begin;
    while (cur < stop) {
      const Span<kTile> span = span_of(p, w.rq, w.rt * kRows);
      w.tiles = span.tiles;
      w.i0 = int(cur - w.item_at), w.i1 = int(min((long long)w.tiles, stop - w.item_at));
      const long long r0 = w.rt * kRows, rows = (long long)w.rq.rows * p.G;
      const int n_rows = int(min((long long)kRows, rows - r0)), base = w.rq.len - w.rq.rows;
      const int first_pos = base + int(r0 / p.G), last_pos = base + int((r0 + n_rows - 1) / p.G);

      // ---- the item's rows: fp16, scaled, in the order of the codes' pairs
      for (int r = warp; r < kRows; r += kWarps) {
        constexpr int kChunks = D / 8;           // 16-byte chunks of eight elements
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < n_rows && lane < kChunks) {
          const long long tok = w.rq.row0 + (r0 + r) / p.G;
          x = __ldg(reinterpret_cast<const uint4*>(p.q + tok * p.q_token +
                                                   (long long)(w.h * p.G + int((r0 + r) % p.G)) * p.q_head) + lane);
        }
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
        float v[8], top = 0.f, sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = DType<T>::to_float(uint16_t(u[e >> 1] >> (16 * (e & 1))));
          top = fmaxf(top, fabsf(v[e])), sum += v[e];
        }
        for (int o = 16; o; o >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        const int ex = int(__float_as_uint(top) >> 23);
        const int fe = ex == 255 || top == 0.f ? 127 : max(24, min(254, 127 + 13 + 127 - ex));   // 2^24 / f stays finite
        const float f = __uint_as_float(uint32_t(fe) << 23), fs = p.scale < 0.f ? -f : f;
        if (lane < kChunks) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float g = e & 1 ? fs * 0.0625f : fs;
            o[e] = half2_of(make_float2(v[e] * g, v[e + 4] * g));
          }
          sts128(sm + S::kQ + (lane >> 3) * (kRows * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
        }
        if (lane == 0) row_k[r] = make_float2(fmaxf(fabsf(p.scale) * (16777216.f / f), 1.17549435e-38f), sum * fs * 5.9604645e-8f);
      }
      tc::fence_proxy_async();
      __syncthreads();

      const Item item{span, r0, n_rows, base, first_pos, last_pos, n, w.i1 - w.i0};
      body(item);
      n += uint32_t(item.count);
      cur = w.item_at + w.i1;
      // ---- on to the next item: the rows' operand and O are free once every role is through
      if (cur < stop) {
        w.item_at += w.tiles;
        if ((w.rt + 1) * kRows < rows) {
          ++w.rt;
        } else {
          w.rt = 0;
          if (++w.h == p.c.heads) {
            w.h = 0;
            do w.rq = tiles_request(p, ++w.b);
            while (w.rq.rows == 0);
          }
        }
      }
      __syncthreads();
      tc::fence_after_sync();
    }
  };

  if (warp < kValueWarp) {
    // ================================================================ softmax: two threads a row
    const int r = tid & 127, half = warp >> 2;
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    items([&](const Item& it) {
      const float2 rk = row_k[r];
      const float2 qf = make_float2(rk.x, rk.x), qs = make_float2(rk.y, rk.y);
      const int pos = r < it.n_rows ? it.base + int((it.r0 + r) / p.G) : -1;
      float m_run = -INFINITY, sig_run = 0.f;
      float2 l2 = make_float2(0.f, 0.f), pm2 = make_float2(0.f, 0.f);
      for (int t = 0; t < it.count; ++t) {
        const uint32_t m = it.n0 + uint32_t(t);
        const int ps = int(m % kParamStages), first = it.span.id(w.i0 + t) * kTile + 64 * half;
        wait(kPrmFull + ps, (m / kParamStages) & 1u, tc::kStatusWaitFull);
        wait(kSFull + int(m & 1), (m >> 1) & 1u, tc::kStatusWaitDone);
        tc::fence_after_sync();
        const uint32_t s_at = lane_base + 256 + 128 * (m & 1);
        const float4* prm = reinterpret_cast<const float4*>(raw_sm + base_off + S::kParam + ps * S::kParamBytes) + 32 * half;
        const uint32_t mine = s_at + 64 * half;
        const bool whole = info[ps].whole != 0;
        uint32_t mask[2] = {0xffffffffu, 0xffffffffu};
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u; };
            const int f = first + 32 * c;
            mask[c] = below(pos + 1 - f) & info[ps].valid[2 * half + c];
            if (p.window) mask[c] &= ~below(pos - p.window + 1 - f) | below(p.sinks - f);
          }
        }
        auto score = [&](float4 k, uint32_t s0, uint32_t s1) {
          return fma2(make_float2(k.x, k.y), make_float2(__uint_as_float(s0), __uint_as_float(s1)),
                      mul2(make_float2(k.z, k.w), qs));
        };
        const float sig_new = info[ps].sig;
        // O times `ab`, each of the two threads half of the row; the products in flight have to be through
        auto rescale = [&](float ab) {
          wait_pv(m - 1);
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[16];
            const uint32_t at = lane_base + half * (D / 2) + 16 * c;
            tc::tmem_ld_32x32b_x16(at, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ab);
            tmem_st16(at, o);
          }
          tc::wait_st();
        };
        bool done = false;
        if (whole && t > 0 && __all_sync(0xffffffffu, m_run > -INFINITY || r >= it.n_rows)) {
          // One pass under the maximum so far, P kept in registers: it holds unless a score is more than 2^8 above.
          const float2 off2 = make_float2(-m_run, -m_run);
          const float2 l_old = l2, pm_old = pm2;
          float top = -INFINITY;
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t s[16];
            tc::tmem_ld_32x32b_x16(mine + 16 * c, s);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 x = fma2(score(prm[8 * c + e], s[2 * e], s[2 * e + 1]), qf, off2);
              top = max3(top, x.x, x.y);
              const float4 v = prm[64 + 8 * c + e];
              const float2 w2 = make_float2(ex2(x.x), ex2(x.y));
              l2 = add2(l2, w2);
              pm2 = fma2(w2, make_float2(v.z, v.w), pm2);
              pk[8 * c + e] = half2_of(mul2(w2, make_float2(v.x, v.y)));
            }
          }
          half_top[m & 1][half][r] = top;
          pair_sync(1 + (warp & 3));
          top = fmaxf(top, half_top[m & 1][half ^ 1][r]);
          done = !__any_sync(0xffffffffu, top > kLazy && r < it.n_rows);
          if (done) {
            if (sig_new != sig_run) rescale(sig_run / sig_new), sig_run = sig_new;
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_st16(mine + 16 * c, reinterpret_cast<const uint32_t(&)[16]>(pk[16 * c]));
          } else {
            l2 = l_old, pm2 = pm_old;
            pair_sync(1 + (warp & 3));           // half_top is written again
          }
        }
        if (!done) {
          // Two passes over 16 tokens at a time, the scores read from tensor memory in each.
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[16];
            tc::tmem_ld_32x32b_x16(mine + 16 * c, s);
            tc::wait_ld();
            const uint32_t see = mask[c >> 1] >> (16 * (c & 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 y = score(prm[8 * c + e], s[2 * e], s[2 * e + 1]);
              if ((see >> (2 * e)) & 1u) top = fmaxf(top, y.x);
              if ((see >> (2 * e + 1)) & 1u) top = fmaxf(top, y.y);
            }
          }
          half_top[m & 1][half][r] = top;
          pair_sync(1 + (warp & 3));
          top = fmaxf(top, half_top[m & 1][half ^ 1][r]) * qf.x;
          if (__any_sync(0xffffffffu, top > m_run + kLazy || sig_new != sig_run)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = m_new == -INFINITY ? 1.f : ex2(m_run - m_new);
            const float ab = alpha * (sig_run / sig_new);
            m_run = m_new, sig_run = sig_new;
            l2 = mul2(l2, make_float2(alpha, alpha));
            pm2 = mul2(pm2, make_float2(alpha, alpha));
            if (t > 0) rescale(ab);
          }
          const float off = m_run == -INFINITY ? 0.f : -m_run;
          const float2 off2 = make_float2(off, off);
          // P of a half lies at the head of that half's scores: columns that this thread has read by then
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[16], pk[8];
            tc::tmem_ld_32x32b_x16(mine + 16 * c, s);
            tc::wait_ld();
            const uint32_t see = mask[c >> 1] >> (16 * (c & 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 x = fma2(score(prm[8 * c + e], s[2 * e], s[2 * e + 1]), qf, off2);
              float4 v = prm[64 + 8 * c + e];
              float2 w2 = make_float2(ex2(x.x), ex2(x.y));
              if (!((see >> (2 * e)) & 1u)) w2.x = v.x = v.z = 0.f;        // what is hidden may be poisoned
              if (!((see >> (2 * e + 1)) & 1u)) w2.y = v.y = v.w = 0.f;
              l2 = add2(l2, w2);
              pm2 = fma2(w2, make_float2(v.z, v.w), pm2);
              pk[e] = half2_of(mul2(w2, make_float2(v.x, v.y)));
            }
            tmem_st8(mine + 8 * c, pk);
          }
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(bar(kPFull + int(m & 1)));
          tc::mbar_arrive(bar(kPrmEmpty + ps));
        }
      }
      // ---- the item's result; each of the two threads writes half of the row
      const uint32_t last = it.n0 + uint32_t(it.count) - 1;
      wait_pv(last);
      tc::fence_after_sync();
      float l = l2.x + l2.y, pm = pm2.x + pm2.y;
      if (half) half_sum[r] = make_float2(l, pm);
      pair_sync(1 + (warp & 3));
      if (!half) {
        l += half_sum[r].x, pm += half_sum[r].y;
        half_sum[r] = make_float2(l, pm);
      }
      pair_sync(1 + (warp & 3));
      l = half_sum[r].x, pm = half_sum[r].y;
      const float back = 16777216.f * sig_run, inv = l == 0.f ? 0.f : 1.f / l;
      const bool starts = w.i0 == 0, ends = w.i1 == w.tiles;
      const long long slot = 2LL * blockIdx.x + (starts ? 1 : 0);
      const long long tok = w.rq.row0 + (it.r0 + r) / p.G;
      const int head = w.h * p.G + int((it.r0 + r) % p.G);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[16];
        const int d = half * (D / 2) + 16 * c;
        tc::tmem_ld_32x32b_x16(lane_base + d, o);
        tc::wait_ld();
        if (r < it.n_rows) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = fmaf(__uint_as_float(o[e]), back, pm);
          if (starts && ends) {
            uint4* to = reinterpret_cast<uint4*>(p.out + tok * p.out_token + (long long)head * p.out_head + d);
            const uint4* gt = reinterpret_cast<const uint4*>(p.gate + tok * p.gate_token + (long long)head * p.gate_head + d);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 gv = p.gate ? __ldg(gt + e) : make_uint4(0, 0, 0, 0);
              const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
              uint32_t out[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                float a = x[8 * e + 2 * k] * inv, b = x[8 * e + 2 * k + 1] * inv;
                if (p.gate) {
                  a /= 1.f + __expf(-DType<T>::to_float(uint16_t(gw[k] & 0xFFFFu)));
                  b /= 1.f + __expf(-DType<T>::to_float(uint16_t(gw[k] >> 16)));
                }
                out[k] = uint32_t(DType<T>::from_float(a)) | (uint32_t(DType<T>::from_float(b)) << 16);
              }
              to[e] = make_uint4(out[0], out[1], out[2], out[3]);
            }
          } else {
            float4* to = reinterpret_cast<float4*>(p.part_o + (slot * kRows + r) * D + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
          }
        }
      }
      if (!(starts && ends) && !half) p.part_ml[slot * kRows + r] = make_float2(m_run, l);
      if (starts && !ends && tid == 0)
        p.meta[blockIdx.x] = make_int4(int((w.item_at + w.tiles - 1) / share), w.b, w.h, int(w.rt));
      tc::fence_before_sync();
    });
  } else if (warp < kKeyWarp) {
    // ================================================================ values: 32 tokens a warp
    const int q = warp - kValueWarp, tg = lane >> 3, g = lane & 7;
    constexpr int kBlocks = D / 64;              // 16-byte loads per lane and 16 tokens
    const int page_mask = (1 << p.c.page_log2) - 1;
    // where the pair of element (n + g) % 8 goes: row, chunk of the swizzle, half of the chunk; a step of 16 tokens
    // flips bit 1 of the chunk
    uint32_t put[8];
    {
      const int tok = 32 * q + 4 * tg;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const uint32_t dim = uint32_t(n + g) & 7u;
        put[n] = sm + S::kV + (tok >> 6) * (D * 128) + (8 * g + dim) * 128 + ((((tok & 63) >> 3) ^ dim) << 4) + (tg & 1) * 8;
      }
    }
    items([&](const Item& it) {
      uint4 vc[kBlocks];                         // the next 16 tokens'
      const uint4 *from[2], *next;
      bool ok[2], next_ok;
      auto locate = [&](int t) {
        const uint32_t m = it.n0 + uint32_t(t);
        const int ps = int(m % kParamStages), first = it.span.id(w.i0 + t) * kTile + 32 * q;
        wait(kPrmFull + ps, (m / kParamStages) & 1u, tc::kStatusWaitFull);
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const int page = info[ps].page[2 * q + blk];
          ok[blk] = unsigned(page) < unsigned(p.c.n_pages);      // after a wait that gave up it may be anything
          from[blk] = reinterpret_cast<const uint4*>(p.c.v + cache_codes_at(ok[blk] ? page : 0, w.h, p.c.heads, p.c.page_log2, D) +
                                                     value_word_at((first + 16 * blk) & page_mask, 0, D)) + lane;
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(kPrmEmpty + ps));
      };
      auto load = [&](int i) { vc[i] = next_ok ? __ldg(next + 32 * i) : make_uint4(0, 0, 0, 0); };
      locate(0);
      next = from[0], next_ok = ok[0];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) load(i);
      for (int t = 0; t < it.count; ++t) {
        const uint32_t m = it.n0 + uint32_t(t), use = m / S::kStages;
        const int st = int(m % S::kStages), vb = 2 * st + (q >> 1);
        if (use > 0) wait(kVEmpty + vb, (use - 1) & 1u, tc::kStatusWaitEmpty);
#pragma unroll 1
        for (int blk = 0; blk < 2; ++blk) {
          if (blk == 0) {
            next = from[1], next_ok = ok[1];
          } else if (t + 1 < it.count) {
            locate(t + 1);
            next = from[0], next_ok = ok[0];
          } else {
            next_ok = false;
          }
          uint32_t to[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) to[n] = (put[n] ^ uint32_t(32 * blk)) + st * S::kOperand;
#pragma unroll
          for (int db = 0; db < kBlocks; ++db) {
            const uint32_t a0 = __funnelshift_r(vc[db].x, vc[db].x, 4 * g), a1 = __funnelshift_r(vc[db].y, vc[db].y, 4 * g);
            const uint32_t a2 = __funnelshift_r(vc[db].z, vc[db].z, 4 * g), a3 = __funnelshift_r(vc[db].w, vc[db].w, 4 * g);
            load(db);                            // into the registers just read
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              uint32_t x = __byte_perm(a0, a1, hf ? 0x7632 : 0x5410), y = __byte_perm(a2, a3, hf ? 0x7632 : 0x5410);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t at = to[hf * 4 + e] + db * 8192;
                if (e & 1) {
                  sts64(at, hfma2(x & 0x00F000F0u, 0x2C002C00u, 0x80088008u), hfma2(y & 0x00F000F0u, 0x2C002C00u, 0x80088008u));
                  x >>= 8, y >>= 8;
                } else {
                  sts64(at, hadd2(x & 0x000F000Fu, 0x80088008u), hadd2(y & 0x000F000Fu, 0x80088008u));
                }
              }
            }
          }
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(kVFull + vb));
      }
    });
  } else if (warp < kParamWarp) {
    // ================================================================ keys: 64 tokens a warp
    // A block of 64 elements is two 16-byte pieces a token: load i holds piece l8 & 1 of token 16 i + tok0.
    const int q = warp - kKeyWarp, l8 = lane >> 3, tk = lane & 7, tok0 = 8 * (l8 >> 1) + tk;
    const int page_mask = (1 << p.c.page_log2) - 1;
    uint32_t put[4];                             // word j of the piece
#pragma unroll
    for (int j = 0; j < 4; ++j) put[j] = sm + S::kK + (64 * q + tok0) * 128 + ((((l8 & 1) * 4 + j) ^ tk) << 4);
    items([&](const Item& it) {
      const int units = it.count * kKB;          // blocks of the item's tiles
      uint4 kc[2][4];                            // the next two blocks
      const uint8_t* from[4];
      bool ok[4];
      auto load = [&](uint4 (&to)[4], int u) {
        if (u % kKB == 0) {
          const uint32_t m = it.n0 + uint32_t(u / kKB);
          const int ps = int(m % kParamStages), first = it.span.id(w.i0 + u / kKB) * kTile + 64 * q + tok0;
          wait(kPrmFull + ps, (m / kParamStages) & 1u, tc::kStatusWaitFull);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int page = info[ps].page[4 * q + i];
            ok[i] = unsigned(page) < unsigned(p.c.n_pages);      // after a wait that gave up it may be anything
            from[i] = p.c.k + cache_codes_at(ok[i] ? page : 0, w.h, p.c.heads, p.c.page_log2, D) +
                      key_word_at((first + 16 * i) & page_mask, 4 * (l8 & 1), D);
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(bar(kPrmEmpty + ps));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          to[i] = ok[i] ? __ldg(reinterpret_cast<const uint4*>(from[i] + 32 * (u % kKB))) : make_uint4(0, 0, 0, 0);
      };
      auto unpack = [&](const uint4 (&c)[4], int u) {
        const uint32_t m = it.n0 + uint32_t(u / kKB), use = m / S::kStages;
        const int st = int(m % S::kStages), kb = u % kKB, kbar = st * kKB + kb;
        if (use > 0) wait(kKEmpty + kbar, (use - 1) & 1u, tc::kStatusWaitEmpty);
        const uint32_t at = uint32_t(st * S::kOperand + kb * (kTile * 128));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = v[j], y = x >> 8;
            sts128(put[j] + at + i * 2048, x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u);
          }
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(kKFull + kbar));
      };
      load(kc[0], 0);
      if (units > 1) load(kc[1], 1);
#pragma unroll 1
      for (int u = 0; u < units; u += 2) {
        unpack(kc[0], u);
        if (u + 2 < units) load(kc[0], u + 2);
        if (u + 1 < units) unpack(kc[1], u + 1);
        if (u + 3 < units) load(kc[1], u + 3);
      }
    });
  } else if (warp == kParamWarp) {
    // ================================================================ parameters: tokens 32 j + lane
    const int page_mask = (1 << p.c.page_log2) - 1;
    items([&](const Item& it) {
      const int* table = p.table + (long long)w.b * p.table_ld;
      float sig = 0.f;                           // running power of two of the item
      int page[4], page_next[4];                 // this tile's, the next one's
      uint32_t kp[4], vp[4];                     // pairs of this tile
      auto pages = [&](int t, int (&to)[4]) {
        const int first = it.span.id(w.i0 + t) * kTile;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = first + 32 * j + lane;
          to[j] = tok < w.rq.len ? table[tok >> p.c.page_log2] : -1;
        }
      };
      auto seen = [&](int tok, int pg) {
        return pg >= 0 && tok <= it.last_pos && (p.window == 0 || tok > it.first_pos - p.window || tok < p.sinks);
      };
      auto pairs = [&](int t) {                  // checks the pages too
        const int first = it.span.id(w.i0 + t) * kTile;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = first + 32 * j + lane;
          if (tok < w.rq.len && unsigned(page[j]) >= unsigned(p.c.n_pages)) {
            atomicExch(&g_tiles_status, kBadPage);
            page[j] = -1;
          }
          kp[j] = vp[j] = 0;
          if (seen(tok, page[j])) {
            const long long at = cache_pair_at(page[j], w.h, p.c.heads, p.c.page_log2, tok & page_mask);
            kp[j] = __ldg(p.c.k_pair + at), vp[j] = __ldg(p.c.v_pair + at);
          }
        }
      };
      pages(0, page);
      pairs(0);
      if (it.count > 1) pages(1, page_next);
      for (int t = 0; t < it.count; ++t) {
        const uint32_t m = it.n0 + uint32_t(t);
        const int ps = int(m % kParamStages), first = it.span.id(w.i0 + t) * kTile;
        float2 kk[4], vv[4];
        float top = kMinStep;
        uint32_t valid[4];
        bool all = true;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kk[j] = lo_step<T>(kp[j]), vv[j] = lo_step<T>(vp[j]);
          valid[j] = __ballot_sync(0xffffffffu, seen(first + 32 * j + lane, page[j]));
          all = all && valid[j] == 0xffffffffu;
          top = fmaxf(top, vv[j].y);
        }
        int now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) now[j] = page[j], page[j] = page_next[j];
        if (t + 1 < it.count) pairs(t + 1);      // under way while this tile's are written
        if (t + 2 < it.count) pages(t + 2, page_next);
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        sig = fmaxf(sig, pow2_above(top));
        const float inv = 1.f / sig;
        if (m >= kParamStages) wait(kPrmEmpty + ps, (m / kParamStages - 1) & 1u, tc::kStatusWaitEmpty);
        float* prm = reinterpret_cast<float*>(raw_sm + base_off + S::kParam + ps * S::kParamBytes);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 32 * j + lane, at = (c >> 1) * 4 + (c & 1);
          prm[at] = kk[j].y, prm[at + 2] = kk[j].x;
          prm[256 + at] = vv[j].y * inv, prm[256 + at + 2] = fmaf(8.f, vv[j].y, vv[j].x);
          if ((lane & 15) == 0) info[ps].page[2 * j + (lane >> 4)] = now[j];
        }
        if (lane == 0) {
          info[ps].sig = sig;
#pragma unroll
          for (int j = 0; j < 4; ++j) info[ps].valid[j] = valid[j];
          info[ps].whole = all && first + kTile <= it.first_pos + 1 &&
                           (p.window == 0 || first > it.last_pos - p.window || first + kTile <= p.sinks);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(kPrmFull + ps));
      }
    });
  } else {
    // ================================================================ products
    items([&](const Item& it) {
      if (tc::elect_one()) {
        const uint64_t tmpl = tc::smem_desc(0u, 16u, 1024u, 2u);
        const uint32_t idesc_s = tc::instr_desc(0, 128, kTile), idesc_o = tc::instr_desc(0, 128, D);
        auto scores = [&](uint32_t m) {
          const int st = int(m % S::kStages);
          // S's buffer held P of the tile before last: its product has to be through
          if (m >= 2 + it.n0) wait_pv(m - 2);
          const uint64_t a = tmpl | ((sm + S::kQ) >> 4), b = tmpl | ((sm + S::kK + st * S::kOperand) >> 4);
#pragma unroll 1
          for (int kb = 0; kb < kKB; ++kb) {
            wait(kKFull + st * kKB + kb, (m / S::kStages) & 1u, tc::kStatusWaitFull);
            tc::fence_after_sync();
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(tmem + 256 + 128 * (m & 1), a + kb * 1024 + k * 2, b + kb * 1024 + k * 2, idesc_s, kb > 0 || k > 0);
            tc::mma_commit(bar(kKEmpty + st * kKB + kb));
          }
          tc::mma_commit(bar(kSFull + int(m & 1)));
        };
        scores(it.n0);
        for (int t = 0; t < it.count; ++t) {
          const uint32_t m = it.n0 + uint32_t(t);
          if (t + 1 < it.count) scores(m + 1);
          const int st = int(m % S::kStages);
          wait(kPFull + int(m & 1), (m >> 1) & 1u, tc::kStatusWaitFull);
          const uint64_t b = tmpl | ((sm + S::kV + st * S::kOperand) >> 4);
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            wait(kVFull + 2 * st + k, (m / S::kStages) & 1u, tc::kStatusWaitFull);
            tc::fence_after_sync();
            tc::mma_ts_kblock(tmem, tmem + 256 + 128 * (m & 1) + 64 * k, uint32_t(b) + k * (D * 8), uint32_t(b >> 32), idesc_o,
                              t > 0 || k > 0);
            tc::mma_commit(bar(kVEmpty + 2 * st + k));
          }
          tc::mma_commit(bar(kPvDone + int(m & 1)));
        }
      }
      __syncwarp();
    });
  }
  if (*abort_flag) {            // a wait gave up: products under way still read shared memory, for microseconds
    const long long t0 = clock64();
    while (clock64() - t0 < 400000) {
    }
    __syncthreads();
  }
  if (warp == kProductWarp) tc::tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int launch(const AttendParams& p, int blocks, cudaStream_t st) {
  static bool configured[64] = {false};
  int dev = 0;
  B200LUT_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    B200LUT_CUDA_OK(cudaFuncSetAttribute(attend_tiles_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem));
    if (dev < 64) configured[dev] = true;
  }
  attend_tiles_kernel<T, D><<<unsigned(blocks), kThreads, Shape<D>::kSmem, st>>>(p);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}

}  // namespace

int attend_tiles_status_take() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_tiles_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_tiles_status, &zero, sizeof(int));
  return v == kBadPage || v == 0 ? v : 0x6300 + v;
}

int attend_tiles(const AttendParams& p, int dtype, int blocks, cudaStream_t st) {
  const bool bf = dtype == B200LUT_BF16;
  switch (p.c.D) {
    case 64: return bf ? launch<__nv_bfloat16, 64>(p, blocks, st) : launch<__half, 64>(p, blocks, st);
    case 128: return bf ? launch<__nv_bfloat16, 128>(p, blocks, st) : launch<__half, 128>(p, blocks, st);
    default: return bf ? launch<__nv_bfloat16, 256>(p, blocks, st) : launch<__half, 256>(p, blocks, st);
  }
}

}  // namespace b200lut
