// Rotary positions over several axes, with an optional RMS norm of every head in front.
//
//   x <- x * rsqrt(mean(x^2) + eps) * gain                               (only with a gain)
//   (x_i, x_{i+R/2}) <- (x_i cos a - x_{i+R/2} sin a, x_{i+R/2} cos a + x_i sin a)     i < R/2
//   a = 2 pi * pos[axis(i), t] * turns(i),  turns(i) = theta^(-2i/R) / (2 pi)
//
// The number of turns is a 64-bit product whose whole part is dropped before it becomes a 32-bit
// angle: at position 2^20 a 32-bit product would be off by 2^-4 turns, this one by 2^-33. The rest is
// fp32, one rounding at the end.
//
// Bound by memory: every element is read and written once. A head's row is D/8 lanes; a lane holds four elements
// of the first half of the rotated part and their four partners (two 8-byte loads), or eight elements that pass, so
// that nothing is exchanged. A warp holds 256/D rows at a time; it computes its token's R/2 sines once and uses
// them for up to seven groups of rows, whose loads are all in flight before the sines are computed. 8192 tokens of 20
// heads of 256 with gains take 40 us, where the bytes would take 26; 51 with partners fetched by shuffles, 47 with one
// element an instruction, 44 with the head's width as an argument, ten more with registers cut to 64 for eight blocks
// an SM: the rest is issue and the chain of loads, sum, turn and stores that each warp runs once. Without gains, 4093
// tokens of 40 heads of 128: 16 us, the bytes 13.
#include <type_traits>

#include "packed.cuh"

namespace b200lut {
namespace {

struct RotaryParams {
  const uint16_t* x[2];        // q, k
  uint16_t* y[2];
  const uint16_t* gain[2];
  long long token_stride[2], head_stride[2];   // of x, in elements; y is [T, heads, D]
  const void* positions;
  long long pos_stride;
  const double* turns;
  const int* axis;
  int T, Hq, H, D, R;
  int groups;                  // groups of 256/D rows per token
  int chunks;                  // ceil(groups / kUnroll)
  float eps;
  bool pos64;
};

constexpr int kWarps = 4;
constexpr float kHuge = 8.470329e-22f;           // 2^-70

template <typename T, int D, int U>
__global__ void __launch_bounds__(kWarps * 32) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) float2 trig[kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * kWarps + warp;        // T * chunks < 2^31
  const int t = int(item / unsigned(p.chunks)), first = int(item - unsigned(t) * p.chunks) * U;
  if (t >= p.T) return;
  constexpr int lanes = D / 8, per = 32 / lanes;           // lanes of a row: 8, 16 or 32
  const int sub = lane / lanes, at = lane % lanes, heads = p.Hq + p.H;
  const bool turned = at < (p.R >> 3);
  // elements a .. a + 3 and b .. b + 3, partners where the lane turns them
  const int a = turned ? 4 * at : 8 * at, b = turned ? a + (p.R >> 1) : a + 4;

  uint2 xa[U], xb[U];
  const uint16_t* in[2] = {p.x[0] + t * p.token_stride[0] + a, p.x[1] + t * p.token_stride[1] + a};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (first + u) * per + sub;
    xa[u] = xb[u] = make_uint2(0, 0);
    if (h < heads) {
      const uint16_t* x = h < p.Hq ? in[0] + h * p.head_stride[0] : in[1] + (h - p.Hq) * p.head_stride[1];
      xa[u] = __ldg(reinterpret_cast<const uint2*>(x));
      xb[u] = __ldg(reinterpret_cast<const uint2*>(x + (b - a)));
    }
  }
  for (int i = lane; i < p.R / 2; i += 32) {
    const long long e = (long long)p.axis[i] * p.pos_stride + t;
    const double pos = p.pos64 ? double(static_cast<const long long*>(p.positions)[e])
                               : double(static_cast<const int*>(p.positions)[e]);
    const double turn = pos * p.turns[i];
    float s, c;
    sincospif(2.f * float(turn - rint(turn)), &s, &c);
    trig[warp][i] = make_float2(c, s);
  }
  __syncwarp();
  // gains of q's four pairs of elements; the last warps of a token have k's rows too
  float2 gain[4];
  auto gains = [&](int side) {
    const uint2 ga = __ldg(reinterpret_cast<const uint2*>(p.gain[side] + a));
    const uint2 gb = __ldg(reinterpret_cast<const uint2*>(p.gain[side] + b));
    gain[0] = unpack2(ga.x, T()), gain[1] = unpack2(ga.y, T()), gain[2] = unpack2(gb.x, T()), gain[3] = unpack2(gb.y, T());
  };
  if (p.gain[0]) gains(0);
  float2 c[2], s[2];
  if (turned) {
    const float4 lo = *reinterpret_cast<const float4*>(&trig[warp][4 * at]);
    const float4 hi = *reinterpret_cast<const float4*>(&trig[warp][4 * at + 2]);
    c[0] = make_float2(lo.x, lo.z), s[0] = make_float2(lo.y, lo.w);
    c[1] = make_float2(hi.x, hi.z), s[1] = make_float2(hi.y, hi.w);
  }
  bool of_q = true;
  const float share = 1.f / D;
  uint16_t* out[2] = {p.y[0] + (long long)t * p.Hq * D + a, p.y[1] + (long long)t * p.H * D + a};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (first + u) * per + sub;
    float2 v[4] = {unpack2(xa[u].x, T()), unpack2(xa[u].y, T()), unpack2(xb[u].x, T()), unpack2(xb[u].y, T())};
    if (p.gain[0]) {
      float2 q = mul2(v[0], v[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) q = fma2(v[e], v[e], q);
      float sum = q.x + q.y;
#pragma unroll
      for (int o = lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      float r = rsqrtf(fmaf(sum, share, p.eps));
      // squares of elements from 2^60 on pass fp32: such a head's are summed again in units of 2^-70
      if (__builtin_expect(__any_sync(0xffffffffu, sum > 3.4e38f), 0)) {
        float again = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 w = mul2(v[e], make_float2(kHuge, kHuge));
          again = fmaf(w.x, w.x, fmaf(w.y, w.y, again));
        }
#pragma unroll 1
        for (int o = lanes >> 1; o; o >>= 1) again += __shfl_xor_sync(0xffffffffu, again, o);
        if (sum > 3.4e38f) r = rsqrtf(again * share) * kHuge;
      }
      if (of_q && h >= p.Hq) gains(1), of_q = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = mul2(v[e], mul2(make_float2(r, r), gain[e]));
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 ws = mul2(v[e + 2], s[e]);
        const float2 y = fma2(v[e], c[e], make_float2(-ws.x, -ws.y));
        v[e + 2] = fma2(v[e + 2], c[e], mul2(v[e], s[e]));
        v[e] = y;
      }
    }
    if (h < heads) {
      uint16_t* o = h < p.Hq ? out[0] + h * D : out[1] + (h - p.Hq) * D;
      *reinterpret_cast<uint2*>(o) = make_uint2(pack2(v[0], T()), pack2(v[1], T()));
      *reinterpret_cast<uint2*>(o + (b - a)) = make_uint2(pack2(v[2], T()), pack2(v[3], T()));
    }
  }
}

}  // namespace
}  // namespace b200lut

using namespace b200lut;

extern "C" int b200lut_rotary(const b200lut_rotary_args* a, void* stream) {
  B200LUT_REQUIRE(a && a->q && a->k && a->q_out && a->k_out && a->positions && a->turns && a->axis, B200LUT_ERR_INVALID,
                  "rotary: null argument");
  B200LUT_REQUIRE(a->dtype == B200LUT_BF16 || a->dtype == B200LUT_F16, B200LUT_ERR_INVALID,
                  "rotary: dtype must be B200LUT_BF16 or B200LUT_F16");
  B200LUT_REQUIRE(a->D == 64 || a->D == 128 || a->D == 256, B200LUT_ERR_UNSUPPORTED,
                  "rotary: head_dim must be 64, 128 or 256 (got %d)", a->D);
  B200LUT_REQUIRE(a->R >= 16 && a->R <= a->D && a->R % 16 == 0, B200LUT_ERR_UNSUPPORTED,
                  "rotary: rotary_dim must be a multiple of 16 up to head_dim (got %d)", a->R);
  B200LUT_REQUIRE(a->T >= 0 && a->n_heads >= 1 && a->n_kv_heads >= 1 && a->n_heads <= 4096 && a->n_kv_heads <= 4096,
                  B200LUT_ERR_INVALID, "rotary: T >= 0 and 1 to 4096 heads of each kind wanted");
  B200LUT_REQUIRE(!a->q_gain == !a->k_gain, B200LUT_ERR_INVALID, "rotary: q_gain and k_gain come together");
  B200LUT_REQUIRE(a->pos_stride >= 0, B200LUT_ERR_INVALID, "rotary: pos_stride must not be negative");
  B200LUT_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->q_out) && aligned16(a->k_out) &&
                      (!a->q_gain || (aligned16(a->q_gain) && aligned16(a->k_gain))) && a->q_token_stride % 8 == 0 &&
                      a->q_head_stride % 8 == 0 && a->k_token_stride % 8 == 0 && a->k_head_stride % 8 == 0,
                  B200LUT_ERR_ALIGN, "rotary: rows must be 16-byte aligned (pointers and strides)");
  if (a->T == 0) return B200LUT_OK;
  RotaryParams p;
  p.x[0] = static_cast<const uint16_t*>(a->q), p.x[1] = static_cast<const uint16_t*>(a->k);
  p.y[0] = static_cast<uint16_t*>(a->q_out), p.y[1] = static_cast<uint16_t*>(a->k_out);
  p.gain[0] = static_cast<const uint16_t*>(a->q_gain), p.gain[1] = static_cast<const uint16_t*>(a->k_gain);
  p.token_stride[0] = a->q_token_stride, p.token_stride[1] = a->k_token_stride;
  p.head_stride[0] = a->q_head_stride, p.head_stride[1] = a->k_head_stride;
  p.positions = a->positions, p.pos_stride = a->pos_stride, p.pos64 = a->pos64 != 0;
  p.turns = a->turns, p.axis = a->axis;
  p.T = a->T, p.Hq = a->n_heads, p.H = a->n_kv_heads, p.D = a->D, p.R = a->R, p.eps = a->eps;
  const int per = 256 / a->D;
  p.groups = (a->n_heads + a->n_kv_heads + per - 1) / per;
  // few tokens: one group of rows per warp, for latency; many: four or seven, which share the sines (seven where that
  // takes fewer warps: of 20 groups three instead of five: a microsecond in 45)
  const int U = (long long)a->T * p.groups <= 148 * 32 ? 1 : (p.groups + 6) / 7 < (p.groups + 3) / 4 ? 7 : 4;
  p.chunks = (p.groups + U - 1) / U;
  const long long items = (long long)a->T * p.chunks, grid = (items + kWarps - 1) / kWarps;
  B200LUT_REQUIRE(items <= 0x7fffff00LL, B200LUT_ERR_UNSUPPORTED, "rotary: too many rows");
  const cudaStream_t st = cudaStream_t(stream);
  const bool bf = a->dtype == B200LUT_BF16;
  const auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return U == 1   ? (bf ? rotary_kernel<__nv_bfloat16, D, 1> : rotary_kernel<__half, D, 1>)
           : U == 4 ? (bf ? rotary_kernel<__nv_bfloat16, D, 4> : rotary_kernel<__half, D, 4>)
                    : (bf ? rotary_kernel<__nv_bfloat16, D, 7> : rotary_kernel<__half, D, 7>);
  };
  auto* kernel = a->D == 64 ? pick(std::integral_constant<int, 64>()) : a->D == 128 ? pick(std::integral_constant<int, 128>())
                                                                                   : pick(std::integral_constant<int, 256>());
  kernel<<<unsigned(grid), kWarps * 32, 0, st>>>(p);
  B200LUT_CUDA_OK(cudaGetLastError());
  return B200LUT_OK;
}
