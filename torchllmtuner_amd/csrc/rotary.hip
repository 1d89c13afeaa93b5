// Rotary positions for the queries and keys of a layer, alone or with the RMS norm of every head in the same
// pass, and their backward passes.  Per token t and pair i of a head's first R = 2 pairs elements
//
//   a = positions[t] * inv_freq[i]       c = f cos a,  s = f sin a        (f: the attention factor)
//   u' = u c - v s,  v' = v c + u s      (u, v) = elements (i, i + R/2), or (2i, 2i + 1) interleaved
//
// elements from R on pass through.  With the norm, x is first x r w with r = rsqrt(mean_d x^2 + eps) of its head.
// Everything in fp32, one rounding to the storage type at the end.  The backward of the rotation is its transpose
// (s -> -s); with g the gradient turned back, gw = g w and xh = x r,
//   dx = r (gw - xh mean_d(gw xh))       dw = sum over tokens and heads of g xh
// and r is formed again from x, which is read anyway: the forward keeps nothing.
//
// Angles: the product of a position and an fp32 frequency has at most 53 bits up to positions of 2^29 and is exact in fp64;
// it is taken to turns with 1/(2 pi) in two fp64 pieces, whole turns go away exactly, and sine and cosine of what is left, at most
// half a turn, are fp32's of its rounded value, turned on by what the rounding took: an angle of a million radians is as good as one of one, and a sine
// near zero as good, relative to itself, as any other.
//
// Bound by HBM: every element is read and written once.  A wave takes one token: its lanes form the token's sines
// and cosines once, a pair a lane, and share them through LDS; then a lane holds the two pieces (16 bytes each where sizes
// and strides allow) whose elements form its pairs, for one head after the other.  The norm's sums run over
// the lanes of a head.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "bf16_tiles.h"
#include "common.h"

namespace mi355 {
namespace {

constexpr int kMaxHead = 512;  // elements of a head
constexpr int kMaxPairs = kMaxHead / 2;

enum { kTurn = 0, kNormTurn = 1, kNormTurnBwd = 2 };

struct QkArgs {
  const void *q, *k;                                       // (T, H, D) and (T, G, D), elements of a head contiguous
  int64_t q_token, q_head, k_token, k_head;                // their strides, in elements
  const void *dq_out, *dk_out;                             // backward with the norm: gradients of the results, dense
  const void *wq, *wk;                                     // (D)
  const void* positions;                                   // (T) int32 or int64
  const float* inv_freq;                                   // (pairs)
  void *oq, *ok;                                           // results, dense (backward: dq and dk, or null)
  float* partial;                                          // backward with the norm: [gridDim.x][2][D] sums of dw, or null
  int64_t T;
  int H, G, D, pairs, wide;                                // wide: positions are int64
  float factor, sign, eps;
  int items, lanes, log_lanes;                             // pairs of pieces a head; lanes a head, a power of two
  int chunks, passes;                                      // waves a token; passes of a wave over heads
};

// N consecutive elements as they lie in memory
template <int BYTES>
struct RawOf;
template <> struct RawOf<2> { typedef uint16_t type; };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<8> { typedef u32x2 type; };
template <> struct RawOf<16> { typedef u32x4 type; };
template <typename T, int N>
using Raw = typename RawOf<N * sizeof(T)>::type;

template <typename T, int N>
__device__ __forceinline__ void widen(const Raw<T, N>& q, float (&v)[N]) {
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (N == 1) {
      v[0] = __uint_as_float(q);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = __uint_as_float(q[j]);
    }
  } else if constexpr (N == 1) {
    v[0] = bf16_to_f32(q);
  } else if constexpr (N == 2) {
    v[0] = __uint_as_float(q << 16);
    v[1] = __uint_as_float(q & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      v[2 * j] = __uint_as_float(q[j] << 16);
      v[2 * j + 1] = __uint_as_float(q[j] & 0xffff0000u);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> narrow(const float (&v)[N]) {
  Raw<T, N> q;
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (N == 1) {
      q = __float_as_uint(v[0]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) q[j] = __float_as_uint(v[j]);
    }
  } else if constexpr (N == 1) {
    q = f32_to_bf16(v[0]);
  } else if constexpr (N == 2) {
    q = pack_bf16x2(v[0], v[1]);
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) q[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
  }
  return q;
}

// the two pieces of an item as u and v of its N pairs, and back: halves lie apart, interleaved pairs side by side
template <int N, bool INTER>
__device__ __forceinline__ void to_pairs(const float (&a)[N], const float (&b)[N], bool turned, float (&u)[N], float (&v)[N]) {
  if constexpr (!INTER || N == 1) {
#pragma unroll
    for (int e = 0; e < N; ++e) u[e] = a[e], v[e] = b[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      u[e] = 2 * e < N ? a[(2 * e) % N] : b[(2 * e) % N];
      v[e] = 2 * e + 1 < N ? a[(2 * e + 1) % N] : b[(2 * e + 1) % N];
    }
  }
}
template <int N, bool INTER>
__device__ __forceinline__ void from_pairs(const float (&u)[N], const float (&v)[N], float (&a)[N], float (&b)[N]) {
  if constexpr (!INTER || N == 1) {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = u[e], b[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      a[e] = e % 2 ? v[e / 2] : u[e / 2];
      b[e] = e % 2 ? v[(N + e) / 2] : u[(N + e) / 2];
    }
  }
}

// sum over groups of `lanes` consecutive lanes, left in all of them
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  auto dpp = [&](auto ctrl) { v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false)); };
  if (lanes > 1) dpp(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  if (lanes > 2) dpp(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  if (lanes > 4) dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (lanes > 8) dpp(std::integral_constant<int, 0x140>{});  // row_mirror
  if (lanes > 16) v += __shfl_xor(v, 16, kWave);
  if (lanes > 32) v += __shfl_xor(v, 32, kWave);
  return v;
}

// cosine and sine, times the factor, of one position and frequency
__device__ __forceinline__ void turn_of(double position, float inv_freq, float factor, float& c, float& s) {
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;  // 1/(2 pi) = kHi + kLo
  const double a = position * static_cast<double>(inv_freq);
  // (one fused operation: a product of its own less the whole turns is one that the compiler may fuse as well, and what it then keeps of the product must
  // not be added a second time)
  const double turns = fma(a, kHi, -rint(a * kHi)) + a * kLo;  // in [-1/2, 1/2]
  const float part = static_cast<float>(turns), rest = static_cast<float>(turns - part) * 6.2831853f;  // (radians, below 2^-23: their square is nothing)
  float sn, cs;
  sincospif(2.0f * part, &sn, &cs);
  c = fmaf(-sn, rest, cs) * factor;
  s = fmaf(cs, rest, sn) * factor;
}

// where the two pieces of item i of a head begin; the second may lie behind the head's end
template <int N, bool INTER>
__device__ __forceinline__ void item_at(int i, int pairs, int& a, int& b, bool& turned) {
  turned = i * N < pairs;
  a = INTER || !turned ? 2 * N * i : N * i;
  b = INTER || !turned ? a + N : a + pairs;
}

template <typename T, int N, int ITER, bool INTER, int MODE>
__global__ __launch_bounds__(256, MODE == kNormTurnBwd ? 4 : 1) void qk_rotary_kernel(const QkArgs p) {
  __shared__ float trig[4][2][kMaxPairs];
  extern __shared__ float dw_sum[];  // kNormTurnBwd: [4][2][D]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = lane >> p.log_lanes, item0 = lane & (p.lanes - 1), heads_pass = kWave >> p.log_lanes;
  const int heads = p.H + p.G;
  int at_a[ITER], at_b[ITER];
  bool has_a[ITER], has_b[ITER], turned[ITER];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int i = item0 + it * p.lanes;
    item_at<N, INTER>(i, p.pairs, at_a[it], at_b[it], turned[it]);
    has_a[it] = i < p.items;
    has_b[it] = has_a[it] && at_b[it] < p.D;
  }
  [[maybe_unused]] float acc_q[ITER][2][N], acc_k[ITER][2][N];
  if constexpr (MODE == kNormTurnBwd) {
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
      for (int e = 0; e < N; ++e) acc_q[it][0][e] = acc_q[it][1][e] = acc_k[it][0][e] = acc_k[it][1][e] = 0.0f;
  }
  const int64_t units = p.T * p.chunks;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave; unit < units; unit += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t t = p.chunks == 1 ? unit : unit / p.chunks;
    const int chunk = p.chunks == 1 ? 0 : static_cast<int>(unit - t * p.chunks);
    const double position = p.wide ? static_cast<double>(static_cast<const int64_t*>(p.positions)[t])
                                   : static_cast<double>(static_cast<const int32_t*>(p.positions)[t]);
    for (int i = lane; i < p.pairs; i += kWave) {
      float c, s;
      turn_of(position, p.inv_freq[i], p.factor, c, s);
      trig[wave][0][i] = c;
      trig[wave][1][i] = s * p.sign;
    }
    wave_lds_sync();
    float c[ITER][N], s[ITER][N];
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = (item0 + it * p.lanes) * N + e;
        c[it][e] = turned[it] ? trig[wave][0][i] : 1.0f;
        s[it][e] = turned[it] ? trig[wave][1][i] : 0.0f;
      }
    wave_lds_sync();  // read by all lanes before the next token's are written
    for (int pass = 0; pass < p.passes; ++pass) {
      const int head = (chunk * p.passes + pass) * heads_pass + sub;
      const bool is_q = head < p.H, on = head < heads;
      const int h = is_q ? head : head - p.H;
      const T* x = is_q ? static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head
                        : static_cast<const T*>(p.k) + t * p.k_token + h * p.k_head;
      const int64_t dense = (t * (is_q ? p.H : p.G) + h) * p.D;
      Raw<T, N> xa[ITER], xb[ITER];
      const Raw<T, N> zero = {};
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        xa[it] = on && has_a[it] ? *reinterpret_cast<const Raw<T, N>*>(x + at_a[it]) : zero;
        xb[it] = on && has_b[it] ? *reinterpret_cast<const Raw<T, N>*>(x + at_b[it]) : zero;
      }
      [[maybe_unused]] Raw<T, N> wa[ITER], wb[ITER], ga[ITER], gb[ITER];
      if constexpr (MODE != kTurn) {
        const T* w = static_cast<const T*>(is_q ? p.wq : p.wk);
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          wa[it] = has_a[it] ? *reinterpret_cast<const Raw<T, N>*>(w + at_a[it]) : zero;
          wb[it] = has_b[it] ? *reinterpret_cast<const Raw<T, N>*>(w + at_b[it]) : zero;
        }
      }
      if constexpr (MODE == kNormTurnBwd) {
        const T* g = static_cast<const T*>(is_q ? p.dq_out : p.dk_out) + dense;
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          ga[it] = on && has_a[it] ? *reinterpret_cast<const Raw<T, N>*>(g + at_a[it]) : zero;
          gb[it] = on && has_b[it] ? *reinterpret_cast<const Raw<T, N>*>(g + at_b[it]) : zero;
        }
      }
      float r = 1.0f;
      if constexpr (MODE != kTurn) {
        float ss = 0.0f;
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          float a[N], b[N];
          widen<T, N>(xa[it], a);
          widen<T, N>(xb[it], b);
#pragma unroll
          for (int e = 0; e < N; ++e) ss += a[e] * a[e] + b[e] * b[e];
        }
        r = 1.0f / sqrtf(lanes_sum(ss, p.lanes) / static_cast<float>(p.D) + p.eps);
      }
      T* out = static_cast<T*>(is_q ? p.oq : p.ok);
      if constexpr (MODE != kNormTurnBwd) {
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          float a[N], b[N], u[N], v[N], u1[N], v1[N];
          widen<T, N>(xa[it], a);
          widen<T, N>(xb[it], b);
          if constexpr (MODE == kNormTurn) {
            float g[N], h2[N];
            widen<T, N>(wa[it], g);
            widen<T, N>(wb[it], h2);
#pragma unroll
            for (int e = 0; e < N; ++e) a[e] = (a[e] * r) * g[e], b[e] = (b[e] * r) * h2[e];
          }
          to_pairs<N, INTER>(a, b, turned[it], u, v);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            u1[e] = u[e] * c[it][e] - v[e] * s[it][e];
            v1[e] = v[e] * c[it][e] + u[e] * s[it][e];
          }
          from_pairs<N, INTER>(u1, v1, a, b);
          // elements that are not turned stay what they are, infinities and NaN payloads of their pair aside
          if constexpr (MODE == kTurn) {
            if (on && has_a[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_a[it]) = turned[it] ? narrow<T, N>(a) : xa[it];
            if (on && has_b[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_b[it]) = turned[it] ? narrow<T, N>(b) : xb[it];
          } else {
            float a0[N], b0[N];
            from_pairs<N, INTER>(u, v, a0, b0);
            if (on && has_a[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_a[it]) = turned[it] ? narrow<T, N>(a) : narrow<T, N>(a0);
            if (on && has_b[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_b[it]) = turned[it] ? narrow<T, N>(b) : narrow<T, N>(b0);
          }
        }
      } else {
        float g0[ITER][N], g1[ITER][N], dot = 0.0f;  // the gradient turned back, as the two pieces
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          float a[N], b[N], u[N], v[N], u1[N], v1[N], xv[N], wv[N];
          widen<T, N>(ga[it], a);
          widen<T, N>(gb[it], b);
          to_pairs<N, INTER>(a, b, turned[it], u, v);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            u1[e] = turned[it] ? u[e] * c[it][e] - v[e] * s[it][e] : u[e];
            v1[e] = turned[it] ? v[e] * c[it][e] + u[e] * s[it][e] : v[e];
          }
          from_pairs<N, INTER>(u1, v1, g0[it], g1[it]);
          widen<T, N>(xa[it], xv);
          widen<T, N>(wa[it], wv);
#pragma unroll
          for (int e = 0; e < N; ++e) dot += (g0[it][e] * wv[e]) * (xv[e] * r);
          widen<T, N>(xb[it], xv);
          widen<T, N>(wb[it], wv);
#pragma unroll
          for (int e = 0; e < N; ++e) dot += (g1[it][e] * wv[e]) * (xv[e] * r);
        }
        const float mean = lanes_sum(dot, p.lanes) / static_cast<float>(p.D);
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
          float xv[N], wv[N], o[N];
          widen<T, N>(xa[it], xv);
          widen<T, N>(wa[it], wv);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float xh = xv[e] * r, d = g0[it][e] * xh;
            o[e] = r * (g0[it][e] * wv[e] - xh * mean);
            acc_q[it][0][e] += on && is_q ? d : 0.0f;
            acc_k[it][0][e] += on && !is_q ? d : 0.0f;
          }
          if (out && on && has_a[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_a[it]) = narrow<T, N>(o);
          widen<T, N>(xb[it], xv);
          widen<T, N>(wb[it], wv);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float xh = xv[e] * r, d = g1[it][e] * xh;
            o[e] = r * (g1[it][e] * wv[e] - xh * mean);
            acc_q[it][1][e] += on && is_q ? d : 0.0f;
            acc_k[it][1][e] += on && !is_q ? d : 0.0f;
          }
          if (out && on && has_b[it]) *reinterpret_cast<Raw<T, N>*>(out + dense + at_b[it]) = narrow<T, N>(o);
        }
      }
    }
  }
  if constexpr (MODE == kNormTurnBwd) {
    if (!p.partial) return;
    // lanes of one item, then the four waves, then (a second kernel) the workgroups: one order, no atomics
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
      for (int e = 0; e < N; ++e)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float a = acc_q[it][half][e], b = acc_k[it][half][e];
          for (int o = p.lanes; o < kWave; o <<= 1) {
            a += __shfl_xor(a, o, kWave);
            b += __shfl_xor(b, o, kWave);
          }
          const bool mine = sub == 0 && (half ? has_b[it] : has_a[it]);
          const int d = (half ? at_b[it] : at_a[it]) + e;
          if (mine) {
            dw_sum[(wave * 2 + 0) * p.D + d] = a;
            dw_sum[(wave * 2 + 1) * p.D + d] = b;
          }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.D; i += 256)
      p.partial[static_cast<int64_t>(blockIdx.x) * 2 * p.D + i] =
          (dw_sum[i] + dw_sum[2 * p.D + i]) + (dw_sum[4 * p.D + i] + dw_sum[6 * p.D + i]);
  }
}

// dw[d] = sum of the workgroups' partial sums: 16 columns x 64 slices a workgroup, the slices added in order
template <typename T>
__global__ __launch_bounds__(1024) void qk_dw_final_kernel(const float* __restrict__ partial, T* __restrict__ dwq,
                                                           T* __restrict__ dwk, int blocks, int D) {
  __shared__ float part[64][17];
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + col;
  float acc = 0.0f;
  if (d < 2 * D) {
#pragma unroll 8
    for (int b = slice; b < blocks; b += 64) acc += partial[static_cast<int64_t>(b) * 2 * D + d];
  }
  part[slice][col] = acc;
  __syncthreads();
  if (slice == 0 && d < 2 * D) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < 64; ++k) total += part[k][col];
    T* out = d < D ? dwq : dwk;
    if (out) store_from_f32(out + (d < D ? d : d - D), total);
  }
}

// Workgroups of the backward with the norm, at most: rows of partial sums, and as many as the card holds at once, four waves a SIMD (with 133 registers
// instead of 128, three, the last quarter waited for the others: 60 us where it is 47 now, 8192 tokens x 36 heads of 128, 4.8 TB/s).
constexpr int kBwdBlocks = 1024;

constexpr int kMostBlocks = 1 << 22;  // of a launch; waves go on to further tokens

// the most elements (16 bytes' worth down to 1) that every piece is a whole number of and starts on
int piece_of(const QkArgs& p, int dtype, std::initializer_list<const void*> ptrs) {
  uintptr_t bits = 0;
  for (const void* x : ptrs) bits |= reinterpret_cast<uintptr_t>(x);
  const int item = dtype == MI355_F32 ? 4 : 2;
  const int64_t sizes = p.pairs | p.D | p.q_token | p.q_head | p.k_token | p.k_head;
  int n = 16 / item;
  while (n > 1 && (sizes % n != 0 || bits % (n * item) != 0)) n /= 2;
  return n;
}

int check_qk(const char* what, const QkArgs& p, int dtype, int64_t H, int64_t G, int64_t D, int64_t pairs) {
  MI355_REQUIRE(dtype == MI355_F32 || dtype == MI355_BF16, "%s: dtype %d is neither fp32 nor bf16", what, dtype);
  MI355_REQUIRE(p.T >= 0 && p.T < (1ll << 31) && H >= 1 && G >= 1 && H + G <= (1 << 16), "%s: bad shape tokens=%lld heads=%lld key heads=%lld",
                what, (long long)p.T, (long long)H, (long long)G);
  MI355_REQUIRE(D >= 2 && D <= kMaxHead, "%s: head size %lld is not within 2 to %d", what, (long long)D, kMaxHead);
  MI355_REQUIRE(pairs >= 1 && 2 * pairs <= D, "%s: %lld frequencies turn more elements than the head's %lld", what, (long long)pairs,
                (long long)D);
  MI355_REQUIRE(std::isfinite(p.factor), "%s: the attention factor must be finite", what);
  return MI355_OK;
}

template <int MODE>
int launch_qk(const char* what, QkArgs p, int dtype, int interleaved, int64_t blocks_at_most, void* stream, int* used) {
  const int n = piece_of(p, dtype, {p.q, p.k, p.oq, p.ok, p.wq, p.wk, p.dq_out, p.dk_out});
  p.items = p.pairs / n + (p.D - 2 * p.pairs + 2 * n - 1) / (2 * n);
  p.lanes = 1, p.log_lanes = 0;
  while (p.lanes < p.items && p.lanes < kWave) p.lanes *= 2, ++p.log_lanes;
  const int heads_pass = kWave / p.lanes, passes = (p.H + p.G + heads_pass - 1) / heads_pass;
  // A wave takes all heads of its token where there are tokens for that many waves; else they are shared out.  Each wave forms the angles again: worth it
  // for what more waves have under way (4096 tokens, 129 heads of 64: 1 wave a token 33.5 us, 8 26.0), but not backward with the norm, whose waves
  // stay for several tokens (8192, 36 of 128: 60 us, with 4 waves a token 71).
  const int64_t want = MODE == kNormTurnBwd ? 4 * kBwdBlocks : 32768;
  const int64_t chunks = p.T >= want ? 1 : std::min<int64_t>(passes, (want + p.T - 1) / p.T);
  p.passes = static_cast<int>((passes + chunks - 1) / chunks);
  p.chunks = (passes + p.passes - 1) / p.passes;
  const int64_t blocks = std::min<int64_t>((p.T * p.chunks + 3) / 4, blocks_at_most);
  if (used) *used = static_cast<int>(blocks);
  const size_t lds = MODE == kNormTurnBwd ? static_cast<size_t>(8) * p.D * sizeof(float) : 0;
  auto run = [&](auto tag, auto pieces) {
    using T = decltype(tag);
    constexpr int N = decltype(pieces)::value;
    constexpr int ITER = N == 1 ? 4 : N == 2 ? 2 : 1;  // (512 elements a head: at most 256, 128 and 64 items of 64 lanes)
    if (interleaved)
      hipLaunchKernelGGL((qk_rotary_kernel<T, N, ITER, true, MODE>), dim3((unsigned)blocks), dim3(256), lds, as_stream(stream), p);
    else
      hipLaunchKernelGGL((qk_rotary_kernel<T, N, ITER, false, MODE>), dim3((unsigned)blocks), dim3(256), lds, as_stream(stream), p);
  };
  const std::integral_constant<int, 1> n1;
  const std::integral_constant<int, 2> n2;
  const std::integral_constant<int, 4> n4;
  const std::integral_constant<int, 8> n8;
  if (dtype == MI355_F32) {
    if (n == 4) run(float{}, n4);
    else if (n == 2) run(float{}, n2);
    else run(float{}, n1);
  } else {
    if (n == 8) run(uint16_t{}, n8);
    else if (n == 4) run(uint16_t{}, n4);
    else if (n == 2) run(uint16_t{}, n2);
    else run(uint16_t{}, n1);
  }
  return check_launch(what);
}

QkArgs qk_args(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head, const void* positions,
               int positions_i64, const float* inv_freq, int64_t pairs, float factor, int64_t T, int64_t H, int64_t G, int64_t D) {
  QkArgs p = {};
  p.q = q, p.k = k, p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head;
  p.positions = positions, p.wide = positions_i64, p.inv_freq = inv_freq, p.factor = factor, p.sign = 1.0f;
  p.T = T, p.H = (int)H, p.G = (int)G, p.D = (int)D, p.pairs = (int)pairs;
  return p;
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                            int64_t k_head_stride, int dtype, const void* positions, int positions_i64, const float* inv_freq,
                            int64_t pairs, float attention_factor, int interleaved, int transpose, void* q_out, void* k_out, int64_t T,
                            int64_t H, int64_t G, int64_t D, void* stream) {
  QkArgs p = qk_args(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, positions, positions_i64, inv_freq, pairs,
                     attention_factor, T, H, G, D);
  if (int rc = check_qk("rotary", p, dtype, H, G, D, pairs)) return rc;
  if (T == 0) return MI355_OK;
  MI355_REQUIRE(q && k && positions && inv_freq && q_out && k_out, "rotary: null pointer");
  p.sign = transpose ? -1.0f : 1.0f;
  p.oq = q_out, p.ok = k_out;
  return launch_qk<kTurn>("rotary", p, dtype, interleaved, kMostBlocks, stream, nullptr);
}

extern "C" int mi355_qk_norm_rotary_fwd(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                        int64_t k_token_stride, int64_t k_head_stride, const void* q_weight, const void* k_weight,
                                        int dtype, const void* positions, int positions_i64, const float* inv_freq, int64_t pairs,
                                        float attention_factor, int interleaved, float epsilon, void* q_out, void* k_out, int64_t T,
                                        int64_t H, int64_t G, int64_t D, void* stream) {
  QkArgs p = qk_args(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, positions, positions_i64, inv_freq, pairs,
                     attention_factor, T, H, G, D);
  if (int rc = check_qk("qk_norm_rotary_fwd", p, dtype, H, G, D, pairs)) return rc;
  MI355_REQUIRE(epsilon >= 0.0f && epsilon < INFINITY, "qk_norm_rotary_fwd: epsilon must be finite and nonnegative");
  if (T == 0) return MI355_OK;
  MI355_REQUIRE(q && k && q_weight && k_weight && positions && inv_freq && q_out && k_out, "qk_norm_rotary_fwd: null pointer");
  p.wq = q_weight, p.wk = k_weight, p.eps = epsilon, p.oq = q_out, p.ok = k_out;
  return launch_qk<kNormTurn>("qk_norm_rotary_fwd", p, dtype, interleaved, kMostBlocks, stream, nullptr);
}

extern "C" int64_t mi355_qk_norm_rotary_bwd_workspace_bytes(int64_t D) {
  return D < 1 || D > kMaxHead ? 0 : static_cast<int64_t>(kBwdBlocks) * 2 * D * 4;
}

extern "C" int mi355_qk_norm_rotary_bwd(const void* dq_out, const void* dk_out, const void* q, int64_t q_token_stride,
                                        int64_t q_head_stride, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                        const void* q_weight, const void* k_weight, int dtype, const void* positions,
                                        int positions_i64, const float* inv_freq, int64_t pairs, float attention_factor,
                                        int interleaved, float epsilon, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                        void* workspace, int64_t T, int64_t H, int64_t G, int64_t D, void* stream) {
  QkArgs p = qk_args(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, positions, positions_i64, inv_freq, pairs,
                     attention_factor, T, H, G, D);
  if (int rc = check_qk("qk_norm_rotary_bwd", p, dtype, H, G, D, pairs)) return rc;
  MI355_REQUIRE(epsilon >= 0.0f && epsilon < INFINITY, "qk_norm_rotary_bwd: epsilon must be finite and nonnegative");
  const bool weights = dq_weight || dk_weight;
  MI355_REQUIRE(T == 0 || (q && k && dq_out && dk_out && q_weight && k_weight && positions && inv_freq), "qk_norm_rotary_bwd: null pointer");
  MI355_REQUIRE(!weights || T == 0 || workspace, "qk_norm_rotary_bwd: workspace required for the weights' gradients");
  p.dq_out = dq_out, p.dk_out = dk_out, p.wq = q_weight, p.wk = k_weight, p.eps = epsilon, p.oq = dq, p.ok = dk, p.sign = -1.0f;
  p.partial = weights ? static_cast<float*>(workspace) : nullptr;
  int used = 0;
  if (T > 0)
    if (int rc = launch_qk<kNormTurnBwd>("qk_norm_rotary_bwd", p, dtype, interleaved, kBwdBlocks, stream, &used)) return rc;
  if (!weights) return MI355_OK;
  const dim3 grid((unsigned)((2 * D + 15) / 16));  // (no tokens: the sum over nothing, zeros)
  if (dtype == MI355_F32)
    hipLaunchKernelGGL(qk_dw_final_kernel<float>, grid, dim3(1024), 0, as_stream(stream), p.partial, static_cast<float*>(dq_weight),
                       static_cast<float*>(dk_weight), used, (int)D);
  else
    hipLaunchKernelGGL(qk_dw_final_kernel<uint16_t>, grid, dim3(1024), 0, as_stream(stream), p.partial,
                       static_cast<uint16_t*>(dq_weight), static_cast<uint16_t*>(dk_weight), used, (int)D);
  return check_launch("qk_norm_rotary_bwd");
}
