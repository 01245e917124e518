// Attention over the 4-bit cache for few rows per request (single tokens): mma.sync on codes, split over tokens.
//
// A work item is 8 NT rows (query heads of one key/value head, times new tokens) of one request. Its visible
// tokens are cut into tiles of 16 or 32; all items' tiles form one line that is dealt to the blocks in equal
// contiguous shares, whatever the requests' lengths. The warps of a block take the tiles of its share in turn,
// each with a running maximum and sum of its own, and join in shared memory; items that span blocks are
// joined by a second kernel in the order of the blocks (deterministic, no atomics).
//
// Operands: the tokens are the M = 16 side of mma.m16n8k16, the rows its N = 8 side, so a tile of codes is
// unpacked once and eight rows ride for free.
//   S^T[token, row] = K[token, :] q[row, :]     A = keys: lane (g, t) holds 16 tokens' rows g and g + 8
//   O^T[dim, row]  += V^T[dim, token] P^T       A = values: lane (g, t) holds elements 8 g .. 8 g + 7 of four tokens;
//                                               their codes at c * 2^-22 and c * 2^-18 (kTop: all at c * 2^-18)
// Row s of A stands for token pi(s) = 4 (s / 2 % 4) + s % 2 + 2 (s / 8) of the tile, so that the four tokens of a
// value lane are adjacent in memory; P^T comes out of S^T by two 8 x 8 transposes of half pairs.
// Every lane copies exactly the 16-byte pieces it will read (cp.async into a ring of its own): no barrier in
// the loop.
#include <climits>
#include <type_traits>

#include "attend.cuh"
#include "packed.cuh"

namespace b200lut {
namespace {

__device__ int g_attend_status = 0;
constexpr int kBadPage = 0x6200;
// What an item costs a block besides its tiles, in tiles: reading the rows, filling the ring, joining the warps. Counted
// in the shares: blocks with six short items took twice as long as blocks with one long one.
constexpr int kItemCost = 24;
constexpr float kLazy = 8.f;           // the running maximum may lag by this many powers of two
constexpr uint32_t kOnes = 0x3C003C00u;     // two halves of 1
// Scores and m are held divided by 2^13: the factor between a product of codes and its score, about 2^11 times the row's
// largest element, then stays finite for every row that bf16 holds. The divisions are exact.
constexpr float kScoreUnit = 8192.f;

template <int D, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  // 16-token pieces of a warp's step. Two halve what a step costs besides its products (32 ragged sequences of up to 8192
  // tokens, 8 heads of 64: 44 us against 50), but at 256 elements the loop then has 1100 instructions, more than the
  // scheduler's instruction cache holds: 134 us where one takes 111 (64 sequences, 4 heads).
  static constexpr int kSub = D == 256 ? 1 : 2;
  static constexpr int kTile = 16 * kSub;
  static constexpr int kWarps = 8;
  static constexpr int kBlocks = NT == 1 ? 2 : 1;              // per SM
  static constexpr int kWords = D / 32;                        // 32-bit words of a key row per lane
  static constexpr int kPieces = D >= 128 ? D / 64 : 1;        // 16-byte key pieces per lane and tile
  static constexpr int kPart = 16 * D + 512;                   // bytes of 16 tokens: keys, values, pairs
  static constexpr int kStage = kSub * kPart;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kFold = kRows * (D + 4) * 4;            // a warp's partial result, in its ring's place
  static constexpr int kRing = kStages * kStage > kFold ? kStages * kStage : kFold;
  static constexpr int kQ = NT * D * 16;                       // query fragments
  static constexpr int kSmem = kQ + kWarps * kRing + kRows * 8 + kWarps * kRows * 8;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Tiles of all items of request b (its row tiles are equal but for what they see).
__device__ __forceinline__ Request rows_request(const AttendParams& p, int b) {
  Request r = request_of(p, b);
  if (r.rows * p.G > p.rows_limit) r.rows = 0;        // the tile kernel's
  return r;
}
template <int kRows, int kTile>
__device__ __forceinline__ long long request_tiles(const AttendParams& p, int b) {
  const Request r = rows_request(p, b);
  long long sum = 0;
  const int rows = r.rows * p.G, base = r.len - r.rows;
  for (int r0 = 0; r0 < rows; r0 += kRows)
    sum += Span<kTile>(base + token_of(p, r0), base + token_of(p, min(r0 + kRows, rows) - 1), r.len, p.window, p.sinks).tiles + kItemCost;
  return sum * p.c.heads;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kWarps * 32, Shape<D, NT>::kBlocks)
attend_rows_kernel(const __grid_constant__ AttendParams p) {
  using S = Shape<D, NT>;
  constexpr int kRows = S::kRows, kWarps = S::kWarps, kTile = S::kTile, kSub = S::kSub;
  // Weights are rounded to fp16 for the products: 2^-11 of each, little beside a bf16 result's rounding of 2^-8, but as
  // much as an fp16 result's own. There a second product takes what the rounding left: 0.3 us of 20 (16 sequences behind
  // a window of 4096).
  constexpr bool kSplit = std::is_same<T, __half>::value;
  // The matrix unit aligns the products of a step by the exponents that their operands are written with, and drops what
  // lies 2^-25 below the largest: of a subnormal the bits that it does not have are lost besides. Codes as the low four
  // bits lose what is 2^-6 below (1 + 2^-10 times 15 and 1, measured), so light weights beside a heavy one came out short:
  // over 131072 tokens the error was 1.10 times a bf16 result's rounding and 2.6 times an fp16 one's (64 elements). So
  // values' codes stand two bits higher, 1.01 times, for one shift more a word; for fp16 results all at the mantissa's top
  // (1.00 times), four shifts instead of one. Neither shows in the times (53.4, 94.3 and 24.6 us; all codes at the top for
  // bf16: 55.3 and 97.7). Keys' codes stay: scores of products alike in size lose nothing that shows.
  constexpr bool kTop = kSplit;
  extern __shared__ __align__(128) uint8_t sm[];
  uint16_t* sq = reinterpret_cast<uint16_t*>(sm);
  uint8_t* ring = sm + S::kQ;
  float2* row_k = reinterpret_cast<float2*>(sm + S::kQ + kWarps * S::kRing);     // factor of q.c, scaled sum of q
  float2* warp_ml = row_k + kRows;                                               // [kWarps][kRows]
  __shared__ long long scan[kWarps];
  __shared__ long long first_tile;
  __shared__ int first_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;

  // ---- this block's share of the line of tiles
  long long total = 0, mine_before = 0;
  const int per = (p.B + kWarps * 32 - 1) / (kWarps * 32);
  long long mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < p.B) mine += request_tiles<kRows, kTile>(p, b);
  }
  long long inc = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) scan[warp] = inc;
  if (tid == 0) first_b = p.B;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) mine_before += scan[w];
    total += scan[w];
  }
  mine_before += inc - mine;
  long long share = (total + gridDim.x - 1) / gridDim.x;
  share = max((long long)kWarps, (share + kWarps - 1) / kWarps * kWarps);
  const long long begin = share * blockIdx.x, stop = min(total, begin + share);
  if (begin >= mine_before && begin < mine_before + mine) {
    long long at = mine_before;
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b >= p.B) break;
      const long long n = request_tiles<kRows, kTile>(p, b);
      if (begin < at + n) {
        first_b = b;
        first_tile = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  if (tid == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  // A launch behind the tile kernel's may run beside its end; the join, which waits for this kernel, needs both complete.
  if (begin >= stop) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(ring + warp * S::kRing));
  const uint32_t q_at = uint32_t(__cvta_generic_to_shared(sq)) + lane * 16;
  const int tok0 = 4 * (g >> 1) + (g & 1);       // tokens of this lane's rows g and g + 8: tok0, tok0 + 2
  long long cur = begin, req_at = first_tile;
  for (int b = first_b; cur < stop && b < p.B; ++b) {
    const Request rq = rows_request(p, b);
    const int rows = rq.rows * p.G;
    const int base = rq.len - rq.rows;
    for (int h = 0; h < p.c.heads && cur < stop; ++h) {
      for (int r0 = 0; r0 < rows && cur < stop; r0 += kRows) {
        const int n_rows = min(kRows, rows - r0);
        const int first_pos = base + token_of(p, r0), last_pos = base + token_of(p, r0 + n_rows - 1);
        const Span<kTile> span(first_pos, last_pos, rq.len, p.window, p.sinks);
        // the item's units: its cost, then its tiles
        const int units = span.tiles + kItemCost;
        const int i0 = max(0, int(min((long long)units, cur - req_at)) - kItemCost);
        const int i1 = max(0, int(min((long long)units, stop - req_at)) - kItemCost);
        if (i0 >= i1) {
          req_at += units;
          cur = max(cur, min(req_at, stop));
          continue;
        }

        // ---- the ring (first, so that its copies are under way while the rows are read)
        __syncthreads();
        const int iters = i1 - i0 > warp ? (i1 - i0 - warp + kWarps - 1) / kWarps : 0;
        const int* table = p.table + (long long)b * p.table_ld;
        // this lane's places in the first page's codes and pairs of the head; a page further is `stride` bytes of codes
        const long long head_at = (long long)h << p.c.page_log2;
        const uint8_t* k_at = p.c.k + head_at * (D / 2) + (D == 64 ? tok0 * 32 + t4 * 8 : tok0 * (D / 2) + t4 * 16);
        const uint8_t* v_at = p.c.v + head_at * (D / 2) + (t4 * 8 + g) * 16;
        const uint32_t* kp_at = p.c.k_pair + head_at + tok0;
        const uint32_t* vp_at = p.c.v_pair + head_at + tok0;
        const uint32_t stride = uint32_t(p.c.heads << p.c.page_log2) * (D / 2);      // at most 4096 * 256 * 128
        int pages = -1;              // lane x: the page of 16 tokens x of the next 32 / kSub steps
        uint32_t bad = 0;            // bit of 16 tokens of a stage: their page is not one of the cache
        auto load = [&](int k) {
          if (k < iters) {
            if (k % (32 / kSub) == 0) {
              const int kk = k + lane / kSub;
              pages = -1;
              if (kk < iters) {
                const int first = span.id(i0 + warp + kk * kWarps) * kTile + 16 * (lane % kSub);
                if (first < rq.len) pages = table[first >> p.c.page_log2];
              }
            }
            const int stage = k % S::kStages;
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
              const int page = __shfl_sync(0xffffffffu, pages, (k % (32 / kSub)) * kSub + s);
              const int first = span.id(i0 + warp + k * kWarps) * kTile + 16 * s;
              const uint32_t bit = 1u << (stage * kSub + s);
              if (unsigned(page) < unsigned(p.c.n_pages)) {
                bad &= ~bit;
                const uint64_t codes = uint64_t(uint32_t(page)) * stride + uint32_t(first & ((1 << p.c.page_log2) - 1)) * (D / 2);
                const uint32_t dst = ring_at + stage * S::kStage + s * S::kPart + lane * 16;
                const uint8_t* kp = k_at + codes;
                if constexpr (D == 64) {
                  cp8(dst, kp);
                  cp8(dst + 8, kp + 64);
                } else {
#pragma unroll
                  for (int i = 0; i < S::kPieces; ++i) cp16(dst + i * 512, kp + (i & 1) * D + (i >> 1) * 64);
                }
                const uint8_t* vp = v_at + codes;
#pragma unroll
                for (int i = 0; i < D / 64; ++i) cp16(dst + S::kPieces * 512 + i * 512, vp + i * 512);
                const uint64_t pair = codes / (D / 2);
                const uint32_t pd = dst + 16 * D;
                cp4(pd, kp_at + pair);
                cp4(pd + 4, kp_at + pair + 2);
                cp4(pd + 8, vp_at + pair);
                cp4(pd + 12, vp_at + pair + 2);
              } else {
                bad |= bit;
                // a page that no row sees a token of (behind the window, say) may be anything
                if (lane == 0 && first < rq.len && first <= last_pos &&
                    (p.window == 0 || first_pos < p.window || first + 15 > first_pos - p.window || first < p.sinks))
                  atomicExch(&g_attend_status, kBadPage);
              }
            }
          }
          cp_commit();
        };
#pragma unroll
        for (int k = 0; k < S::kStages - 1; ++k) load(k);

        // ---- the item's rows as fp16 fragments
        for (int r = warp; r < kRows; r += kWarps) {
          constexpr int kChunks = D / 8;         // 16-byte chunks: the eight elements of one word of codes
          uint4 x = make_uint4(0, 0, 0, 0);
          if (r < n_rows && lane < kChunks) {
            const int tok = token_of(p, r0 + r);
            x = __ldg(reinterpret_cast<const uint4*>(p.q + (rq.row0 + tok) * p.q_token +
                                                     (long long)(h * p.G + r0 + r - tok * p.G) * p.q_head) + lane);
          }
          const uint32_t u[4] = {x.x, x.y, x.z, x.w};
          float v[8], top = 0.f, sum = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = DType<T>::to_float(uint16_t(u[e >> 1] >> (16 * (e & 1))));
            top = fmaxf(top, fabsf(v[e])), sum = fmaf(v[e], kSumUnit, sum);
          }
          for (int o = 16; o; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
          }
          const int ex = int(__float_as_uint(top) >> 23);                // exponent of the largest element
          const int fe = ex == 255 || top == 0.f ? 127 : min(254, 127 + 13 + 127 - ex);
          const float f = __uint_as_float(uint32_t(fe) << 23);
          if (lane < kChunks) {
            const int tig = D == 64 ? lane / 2 : (lane % 16) / 4, w = D == 64 ? lane % 2 : (lane / 16) * 4 + lane % 4;
            uint4 o;
            o.x = half2_of(v[0] * f, v[4] * f), o.y = half2_of(v[1] * f * 0.0625f, v[5] * f * 0.0625f);
            o.z = half2_of(v[2] * f, v[6] * f), o.w = half2_of(v[3] * f * 0.0625f, v[7] * f * 0.0625f);
            reinterpret_cast<uint4*>(sq)[((r >> 3) * S::kWords + w) * 32 + (r & 7) * 4 + tig] = o;
          }
          if (lane == 0) row_k[r] = make_float2(p.scale * (16777216.f / kScoreUnit / f), p.scale * sum * (1.f / kScoreUnit / kSumUnit));
        }
        __syncthreads();

        float qf[NT][2], qs[NT][2], m[NT][2], l[NT][2], pm[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + 2 * t4 + e;
            const float2 k = row_k[r];
            qf[n][e] = k.x, qs[n][e] = k.y;
            m[n][e] = -INFINITY, l[n][e] = 0.f, pm[n][e] = 0.f;
          }
        float o[NT][D / 16][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
        float ws[NT][4];             // sums of the rounded weights (every row of A is ones)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) ws[n][e] = 0.f;

        for (int k = 0; k < iters; ++k) {
          cp_wait<S::kStages - 2>();
          const int stage = k % S::kStages;
          const uint32_t missing = bad >> (stage * kSub);
          load(k + S::kStages - 1);
          const uint32_t at = ring_at + stage * S::kStage + lane * 16;

          // ---- scores
          float acc[kSub][NT][2][4];
#pragma unroll
          for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 8; ++i) acc[s][n][i >> 2][i & 3] = 0.f;
          // word w of the rows: x and y are those of the lane's two tokens
          auto qk = [&](int s, uint32_t x, uint32_t y, const uint4 (&q)[NT]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16(acc[s][n][0], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q[n].x, q[n].y);
              mma16(acc[s][n][1], (x >> 8) & 0x000F000Fu, (y >> 8) & 0x000F000Fu, (x >> 8) & 0x00F000F0u,
                    (y >> 8) & 0x00F000F0u, q[n].z, q[n].w);
            }
          };
          auto q_of = [&](uint4 (&q)[NT], int w) {
#pragma unroll
            for (int n = 0; n < NT; ++n) q[n] = lds128(q_at + (n * S::kWords + w) * 512);
          };
          if constexpr (D == 64) {
            uint4 a[kSub], q[NT];
#pragma unroll
            for (int s = 0; s < kSub; ++s) a[s] = lds128(at + s * S::kPart);
            q_of(q, 0);
#pragma unroll
            for (int s = 0; s < kSub; ++s) qk(s, a[s].x, a[s].z, q);
            q_of(q, 1);
#pragma unroll
            for (int s = 0; s < kSub; ++s) qk(s, a[s].y, a[s].w, q);
          } else {
#pragma unroll
            for (int i = 0; i < S::kPieces; i += 2) {
              uint4 a[kSub], c[kSub], q[NT];
#pragma unroll
              for (int s = 0; s < kSub; ++s) a[s] = lds128(at + s * S::kPart + i * 512), c[s] = lds128(at + s * S::kPart + (i + 1) * 512);
              q_of(q, i * 2);
#pragma unroll
              for (int s = 0; s < kSub; ++s) qk(s, a[s].x, c[s].x, q);
              q_of(q, i * 2 + 1);
#pragma unroll
              for (int s = 0; s < kSub; ++s) qk(s, a[s].y, c[s].y, q);
              q_of(q, i * 2 + 2);
#pragma unroll
              for (int s = 0; s < kSub; ++s) qk(s, a[s].z, c[s].z, q);
              q_of(q, i * 2 + 3);
#pragma unroll
              for (int s = 0; s < kSub; ++s) qk(s, a[s].w, c[s].w, q);
            }
          }

          // ---- probabilities
          const int first = span.id(i0 + warp + k * kWarps) * kTile;
          float2 v[kSub][2];                     // lo, step of the lane's two tokens
          float x[kSub][NT][4];
#pragma unroll
          for (int s = 0; s < kSub; ++s) {
            const uint4 pr = lds128(at + s * S::kPart + 16 * D);
            const float2 k0 = lo_step<T>(pr.x), k1 = lo_step<T>(pr.y);
            v[s][0] = lo_step<T>(pr.z), v[s][1] = lo_step<T>(pr.w);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 kk = e < 2 ? k0 : k1;
                x[s][n][e] = fmaf(kk.y, (acc[s][n][0][e] + acc[s][n][1][e]) * qf[n][e & 1], kk.x * qs[n][e & 1]);
              }
          }
          // (first + kTile can be 2^31)
          const bool whole = (missing & ((1u << kSub) - 1u)) == 0 && first <= first_pos + 1 - kTile && first <= rq.len - kTile &&
                             (p.window == 0 || first > last_pos - p.window || first <= p.sinks - kTile);
          uint32_t hidden = 0;
          if (!whole) {
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
              bool seen[2] = {false, false};     // some row of this lane sees the token
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int j = first + 16 * s + tok0 + (e < 2 ? 0 : 2), r = n * 8 + 2 * t4 + (e & 1);
                  const int pos = r < n_rows ? base + token_of(p, r0 + r) : -1;
                  if (!((missing >> s) & 1u) && token_seen(j, pos, rq.len, p.window, p.sinks)) seen[e >> 1] = true;
                  else x[s][n][e] = -INFINITY, hidden |= 1u << ((s * NT + n) * 4 + e);
                }
              // what lies in hidden places may be anything, NaN too
              if (!seen[0]) v[s][0] = make_float2(0.f, 0.f);
              if (!seen[1]) v[s][1] = make_float2(0.f, 0.f);
            }
          }
          float mid[kSub][2], big = kMinStep;    // the lane's largest token
#pragma unroll
          for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mid[s][i] = fmaf(7.5f, v[s][i].y, v[s][i].x);
              big = fmaxf(big, token_size(v[s][i].y, mid[s][i]));
            }
          const float room = (kLazy - size_in_m(big)) * (1.f / kScoreUnit);
          bool grow = false;
#pragma unroll
          for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) grow |= x[s][n][e] > m[n][e & 1] + room;
          if (__any_sync(0xffffffffu, grow)) {
            float size[kSub][2];
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
              for (int i = 0; i < 2; ++i) size[s][i] = size_in_m(token_size(v[s][i].y, mid[s][i])) * (1.f / kScoreUnit);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float top = fmaxf(x[0][n][e] + size[0][0], x[0][n][e + 2] + size[0][1]);
                if constexpr (kSub == 2)
                  top = fmaxf(top, fmaxf(x[kSub - 1][n][e] + size[kSub - 1][0], x[kSub - 1][n][e + 2] + size[kSub - 1][1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float m_new = fmaxf(m[n][e], top);
                const float root = m_new == -INFINITY ? 1.f : ex2(0.5f * kScoreUnit * (m[n][e] - m_new)), alpha = root * root;
                m[n][e] = m_new;
                l[n][e] = l[n][e] * root * root;
                pm[n][e] *= alpha;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[n][i][e] *= alpha, o[n][i][e + 2] *= alpha;
                ws[n][e] *= alpha;
              }
          }
          float off[NT][2];                      // of a score beyond fp32 the weight is infinite or NaN
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) off[n][e] = m[n][e] == -INFINITY ? 0.f : fmaxf(-3e38f, m[n][e] * -kScoreUnit);
          uint32_t bf[kSub][NT][2], rest[kSub][NT][2];
#pragma unroll
          for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float pr = ex2(fmaf(x[s][n][e], kScoreUnit, off[n][e & 1]));
                const bool none = (hidden >> ((s * NT + n) * 4 + e)) & 1u;
                l[n][e & 1] += pr;
                pm[n][e & 1] += none ? 0.f : pr * mid[s][e >> 1];
                w[e] = none ? 0.f : pr * v[s][e >> 1].y;
              }
              const uint32_t h0 = half2_of(w[0], w[1]), h1 = half2_of(w[2], w[3]);
              bf[s][n][0] = transpose8x8(h0);
              bf[s][n][1] = transpose8x8(h1);
              mma16(ws[n], kOnes, kOnes, kOnes, kOnes, bf[s][n][0], bf[s][n][1]);
              if constexpr (kSplit) {
                const float2 f0 = unpack2(h0, __half()), f1 = unpack2(h1, __half());
                rest[s][n][0] = transpose8x8(half2_of(w[0] - f0.x, w[1] - f0.y));
                rest[s][n][1] = transpose8x8(half2_of(w[2] - f1.x, w[3] - f1.y));
                mma16(ws[n], kOnes, kOnes, kOnes, kOnes, rest[s][n][0], rest[s][n][1]);
              }
            }

          // ---- values
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
              const uint4 c = lds128(at + s * S::kPart + S::kPieces * 512 + i * 512);
              const uint32_t x01 = __byte_perm(c.x, c.y, 0x5410), y01 = __byte_perm(c.x, c.y, 0x7632);
              const uint32_t x23 = __byte_perm(c.z, c.w, 0x5410), y23 = __byte_perm(c.z, c.w, 0x7632);
              auto code = [](uint32_t x, int j) {          // code j of each half, high in the mantissa
                if (kTop) return (j == 0 ? x << 6 : j == 1 ? x << 2 : j == 2 ? x >> 2 : x >> 6) & 0x03C003C0u;
                return (j < 2 ? x << 2 : x >> 6) & (j & 1 ? 0x03C003C0u : 0x003C003Cu);
              };
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t a0 = code(x01, j), a1 = code(y01, j), a2 = code(x23, j), a3 = code(y23, j);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma16(o[n][i * 4 + j], a0, a1, a2, a3, bf[s][n][0], bf[s][n][1]);
                  if constexpr (kSplit) mma16(o[n][i * 4 + j], a0, a1, a2, a3, rest[s][n][0], rest[s][n][1]);
                }
              }
            }
        }
        cp_wait<0>();

        // ---- the warps' results joined
        float* fold = reinterpret_cast<float*>(ring + warp * S::kRing);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
              l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], s);
              pm[n][e] += __shfl_xor_sync(0xffffffffu, pm[n][e], s);
            }
            const int r = n * 8 + 2 * t4 + e;
            if (g == 0) warp_ml[warp * kRows + r] = make_float2(m[n][e], l[n][e]);
            const float mid = fmaf(-7.5f, ws[n][e], pm[n][e]);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const float f = kTop || (i & 1) ? 262144.f : 4194304.f;
              const int d = (i >> 2) * 64 + 8 * g + (i & 3);
              fold[r * (D + 4) + d] = fmaf(o[n][i][e], f, mid);
              fold[r * (D + 4) + d + 4] = fmaf(o[n][i][e + 2], f, mid);
            }
          }
        __syncthreads();
        const bool starts = i0 == 0, ends = i1 == span.tiles;
        const long long slot = 2LL * blockIdx.x + (starts ? 1 : 0);
        for (int i = tid; i < n_rows * (D / 2); i += kWarps * 32) {
          const int r = i / (D / 2), d = 2 * (i % (D / 2));
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_ml[w * kRows + r].x);
          float sum = 0.f, a = 0.f, c = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float2 ml = warp_ml[w * kRows + r];
            const float root = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(0.5f * kScoreUnit * (ml.x - top)), f = root * root;
            const float* part = reinterpret_cast<const float*>(ring + w * S::kRing) + r * (D + 4) + d;
            sum = fmaf(ml.y * root, root, sum);
            a = fmaf(part[0], f, a);
            c = fmaf(part[1], f, c);
          }
          if (starts && ends) {
            const int at = token_of(p, r0 + r), head = h * p.G + r0 + r - at * p.G;
            const long long tok = rq.row0 + at;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const uint32_t lo = DType<T>::from_float(gated<T>(a * inv, p, tok, head, d));
            const uint32_t hi = DType<T>::from_float(gated<T>(c * inv, p, tok, head, d + 1));
            *reinterpret_cast<uint32_t*>(p.out + tok * p.out_token + (long long)head * p.out_head + d) = lo | (hi << 16);
          } else {
            *reinterpret_cast<float2*>(p.part_o + (slot * kRows + r) * D + d) = make_float2(a, c);
            if (d == 0) p.part_ml[slot * kRows + r] = make_float2(top * kScoreUnit, sum);
          }
        }
        if (starts && !ends && tid == 0) {
          const long long last = (req_at + units - 1) / share;
          p.meta[blockIdx.x] = joined_item(p, int(last), rq, h, r0, n_rows);
        }
        req_at += units;
        cur = min(req_at, stop);
      }
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// What a kernel left to be joined: `blocks` blocks with items of at most `rows` rows, `per` blocks of the join each.
struct JoinSide {
  const int4* meta;
  const float2* ml;
  const float* o;
  int blocks, rows, per;
};

// Joins the parts of the items that a block began and others went on with. With many parts all warps of a block share a
// row: each adds every eighth part, then the first adds the warps' sums in their order; with few a warp has a row to
// itself.
constexpr int kJoinWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const __grid_constant__ AttendParams p,
                                                                      const JoinSide first_side, const JoinSide second_side) {
  constexpr int kPer = D / 32;
  __shared__ float part[kJoinWarps][D + 2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cut = first_side.blocks * first_side.per;
  const bool second = int(blockIdx.x) >= cut;
  const JoinSide& side = second ? second_side : first_side;
  const int id = int(blockIdx.x) - (second ? cut : 0), c0 = id / side.per, y = id % side.per;
  const int4 meta = side.meta[c0];
  if (meta.x == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_rows = (meta.w & 127) + 1;
  const int c1 = meta.x, ways = c1 - c0 >= 16 ? kJoinWarps : 1, step = kJoinWarps / ways, way = warp / step;
  const int h = meta.w >> 13, rem = (meta.w >> 7) & 63;
  for (int first = y * step; first < n_rows; first += side.per * step) {
    const int r = first + warp % step;
    const bool live = r < n_rows;
    auto slot = [&](int c) { return (c == c0 ? 2LL * c + 1 : 2LL * c) * side.rows + r; };
    float top = -INFINITY, sum = 0.f, x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = 0.f;
    if (live) {
      for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, side.ml[slot(c)].x);
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll 4
      for (int c = c0 + way; c <= c1; c += ways) {
        const float2 ml = side.ml[slot(c)];
        const float* o = side.o + slot(c) * D + lane * kPer;
        float v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          const float2 z = *reinterpret_cast<const float2*>(o + i);
          v[i] = z.x, v[i + 1] = z.y;
        }
        const float root = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(0.5f * (ml.x - top)), f = root * root;
        sum = fmaf(ml.y * root, root, sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = fmaf(v[i], f, x[i]);
      }
    }
    if (ways > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) part[warp][lane * kPer + i] = x[i];
      if (lane == 0) part[warp][D] = sum;
      __syncthreads();
      if (way == 0)
        for (int w = 1; w < ways; ++w) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) x[i] += part[warp + w * step][lane * kPer + i];
          sum += part[warp + w * step][D];
        }
    }
    if (live && way == 0) {
      const int at = token_of(p, rem + r), head = h * p.G + rem + r - at * p.G, d = lane * kPer;
      const long long tok = meta.y + at;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint32_t* to = reinterpret_cast<uint32_t*>(p.out + tok * p.out_token + (long long)head * p.out_head + d);
#pragma unroll
      for (int i = 0; i < kPer; i += 2)
        to[i / 2] = uint32_t(DType<T>::from_float(gated<T>(x[i] * inv, p, tok, head, d + i))) |
                    (uint32_t(DType<T>::from_float(gated<T>(x[i + 1] * inv, p, tok, head, d + i + 1))) << 16);
    }
  }
}

// A launch that may begin before the one in front of it has ended.
template <typename... P>
int launch_behind(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const P&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  B200LUT_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
  return B200LUT_OK;
}

template <typename T, int D, int NT>
int launch(const AttendParams& p, int blocks, bool behind, cudaStream_t st) {
  using S = Shape<D, NT>;
  static bool configured[64] = {false};
  int dev = 0;
  B200LUT_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    B200LUT_CUDA_OK(cudaFuncSetAttribute(attend_rows_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    if (dev < 64) configured[dev] = true;
  }
  if (behind) return launch_behind(attend_rows_kernel<T, D, NT>, unsigned(blocks), S::kWarps * 32, S::kSmem, st, p);
  attend_rows_kernel<T, D, NT><<<unsigned(blocks), S::kWarps * 32, S::kSmem, st>>>(p);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}

// Rows of an item, and of a request that comes with row starts and is still this kernel's (rows_limit): one item's. The
// other side of that limit, measured with up to 8 heads a key head, 64 requests of 4096 to 8192 tokens (a row tile more
// for every 8 rows here against one tile of 128 there): 8 rows 139 us here; 16 rows 242 here and 349 there, 24 rows 343
// and 351, 32 rows 448 and 351 (4 heads of 256); 242 and 519, 351 and 518, 455 and 518, 48 rows 674 and 526 (8 heads of
// 128); 32 requests of one head of 64: 16 rows 31 and 65, 64 rows 59 and 69. So the tile kernel is the better one from some 24,
// 32 and 64 rows on; between 9 rows and there a request costs up to twice what two or three items here would.
int rows_of(int G) { return G <= 8 ? 8 : 16; }
int row_blocks(int sms, int G) { return G <= 8 ? 2 * sms : sms; }      // Shape::kBlocks

// Workspace of a launch over `blocks` blocks of `rows` rows: what attend_*_kernel leave to the join.
size_t workspace_of(int blocks, int rows, int D) { return size_t(blocks) * (16 + 2 * size_t(rows) * (8 + size_t(D) * 4)); }
void lay_out(AttendParams* p, void* ws, int blocks, int rows) {
  p->meta = static_cast<int4*>(ws);
  p->part_ml = reinterpret_cast<float2*>(p->meta + blocks);
  p->part_o = reinterpret_cast<float*>(p->part_ml + 2LL * blocks * rows);
}

template <typename T, int D>
int run(AttendParams p, int sms, void* ws, cudaStream_t st) {
  const int blocks = row_blocks(sms, p.G), rows = rows_of(p.G);
  JoinSide tiles = {nullptr, nullptr, nullptr, 0, 128, 16};
  p.rows_limit = INT_MAX;
  if (p.row_start) {
    // requests of many rows first, on the tensor cores; the others' launch follows on their heels
    p.rows_limit = rows;
    AttendParams t = p;
    lay_out(&t, static_cast<char*>(ws) + workspace_of(blocks, rows, D), sms, 128);
    const int rc = attend_tiles(t, DType<T>::id, sms, st);
    if (rc != B200LUT_OK) return rc;
    tiles.meta = t.meta, tiles.ml = t.part_ml, tiles.o = t.part_o, tiles.blocks = sms;
  }
  lay_out(&p, ws, blocks, rows);
  const bool behind = p.row_start != nullptr;
  const int rc = rows == 8 ? launch<T, D, 1>(p, blocks, behind, st) : launch<T, D, 2>(p, blocks, behind, st);
  if (rc != B200LUT_OK) return rc;
  const JoinSide side = {p.meta, p.part_ml, p.part_o, blocks, rows, 4};
  return launch_behind(attend_join_kernel<T, D>, unsigned(side.blocks * side.per + tiles.blocks * tiles.per), kJoinWarps * 32, 0,
                       st, p, side, tiles);
}

template <typename T>
int pick_dim(const AttendParams& p, int sms, void* ws, cudaStream_t st) {
  return p.c.D == 64 ? run<T, 64>(p, sms, ws, st) : p.c.D == 128 ? run<T, 128>(p, sms, ws, st) : run<T, 256>(p, sms, ws, st);
}

size_t workspace_bytes_of(int G, int D, bool one_row_each, int sms) {
  return workspace_of(row_blocks(sms, G), rows_of(G), D) + (one_row_each ? 0 : workspace_of(sms, 128, D));
}

}  // namespace

int attend_page_take() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attend_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_attend_status, &zero, sizeof(int));
  const int tiles = attend_tiles_page_take();        // one word to the caller
  return v != 0 ? v : tiles;
}

}  // namespace b200lut

using namespace b200lut;

extern "C" size_t b200lut_attend_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int one_row_each) {
  if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  return workspace_bytes_of(n_heads / n_kv_heads, head_dim, one_row_each != 0, b200lut_sm_count());
}

extern "C" int b200lut_attend(const b200lut_attend_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  B200LUT_REQUIRE(a, B200LUT_ERR_INVALID, "attend: null argument");
  AttendParams p = {};
  const int rc = check_cache(a->cache, "attend", &p.c);
  if (rc != B200LUT_OK) return rc;
  B200LUT_REQUIRE(a->T >= 0 && a->B >= 0, B200LUT_ERR_INVALID, "attend: T and B must not be negative");
  B200LUT_REQUIRE(a->n_heads >= 1 && a->n_heads % p.c.heads == 0, B200LUT_ERR_INVALID,
                  "attend: n_heads %d is not a multiple of the cache's %d heads", a->n_heads, p.c.heads);
  B200LUT_REQUIRE(a->n_heads / p.c.heads <= 64, B200LUT_ERR_UNSUPPORTED,
                  "attend: at most 64 query heads per key/value head (got %d)", a->n_heads / p.c.heads);
  B200LUT_REQUIRE(a->window >= 0 && a->sinks >= 0 && a->width >= 1 && a->B <= 65536, B200LUT_ERR_INVALID,
                  "attend: window and sinks must not be negative, width must be positive, B at most 65536");
  B200LUT_REQUIRE(fabsf(a->scale) < 1.7014118e38f, B200LUT_ERR_INVALID, "attend: scale must be finite, below 2^127");
  if (a->T == 0 || a->B == 0) return B200LUT_OK;
  B200LUT_REQUIRE(a->q && a->out && a->block_table && a->kv_len, B200LUT_ERR_INVALID, "attend: null argument");
  B200LUT_REQUIRE(a->row_start || a->T == a->B, B200LUT_ERR_INVALID,
                  "attend: without row_start there is one row per request (T %d, B %d)", a->T, a->B);
  B200LUT_REQUIRE(aligned16(a->q) && aligned16(a->out) && (!a->gate || aligned16(a->gate)) && a->q_token_stride % 8 == 0 &&
                      a->q_head_stride % 8 == 0 && a->out_token_stride % 8 == 0 && a->out_head_stride % 8 == 0 &&
                      (!a->gate || (a->gate_token_stride % 8 == 0 && a->gate_head_stride % 8 == 0)),
                  B200LUT_ERR_ALIGN, "attend: rows must be 16-byte aligned (pointers and strides)");
  const int sms = b200lut_sm_count();
  B200LUT_REQUIRE(workspace && aligned16(workspace) &&
                      workspace_bytes >= workspace_bytes_of(a->n_heads / p.c.heads, p.c.D, !a->row_start, sms),
                  B200LUT_ERR_WORKSPACE, "attend: workspace of b200lut_attend_workspace_bytes() wanted");
  p.q = static_cast<const uint16_t*>(a->q), p.gate = static_cast<const uint16_t*>(a->gate);
  p.out = static_cast<uint16_t*>(a->out);
  p.q_token = a->q_token_stride, p.q_head = a->q_head_stride;
  p.gate_token = a->gate_token_stride, p.gate_head = a->gate_head_stride;
  p.out_token = a->out_token_stride, p.out_head = a->out_head_stride;
  p.table = a->block_table, p.table_ld = a->table_stride, p.kv_len = a->kv_len, p.row_start = a->row_start;
  p.T = a->T, p.B = a->B, p.Hq = a->n_heads, p.G = a->n_heads / p.c.heads, p.width = a->width;
  p.window = a->window, p.sinks = a->sinks;
  B200LUT_REQUIRE((long long)a->T * p.G <= INT_MAX - 256, B200LUT_ERR_UNSUPPORTED, "attend: too many rows (T %d)", a->T);
  int up = 0;                  // 2^up is the power of two >= G
  while ((1 << up) < p.G) ++up;
  p.g_mul = uint32_t(((1ull << (31 + up)) + p.G - 1) / p.G), p.g_shift = up - 1;
  p.scale = a->scale * 1.4426950408889634f;
  p.wait_cycles = gemm_wait_cycles();
  const cudaStream_t st = cudaStream_t(stream);
  return a->cache->dtype == B200LUT_BF16 ? pick_dim<__nv_bfloat16>(p, sms, workspace, st) : pick_dim<__half>(p, sms, workspace, st);
}
