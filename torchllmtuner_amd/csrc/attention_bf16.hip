// Causal attention over packed sequences (attention.h has the formulas) on v_mfma_f32_32x32x16_bf16: bf16 storage, head sizes in whole
// 16-byte pieces up to 256, fp32 sums and statistics.
//
// The matrix instruction takes per lane 8 elements of a row (column) lane % 32 at k = 8 (lane / 32) .. + 7 and yields 16 fp32 of column
// lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4.  Products are formed turned so that a result is the next product's right operand where
// it lies, without a trip through LDS: the forward and dq form s^T = K Q^T, a column a query, so a query's weights lie in its two
// lanes (lane and lane + 32), its maximum and sum are in-lane reductions and one exchange, and o^T += V^T p^T takes
// the weights as they are, rounded to bf16; dk and dv form s = Q K^T, a column a key, for dv^T += dO^T p and dk^T += Q^T ds.
// The keys of 16 then meet in the order in which the result holds them, 4 h + {0..3} and 8 + 4 h + {0..3} for lane half h, which
// only says which rows the left operand's transposing LDS reads fetch.
//
// A wave holds 32 rows (queries, or keys), a workgroup four waves.  The other axis passes through LDS in tiles of 64 rows, requested
// straight into LDS a tile ahead, two buffers, one barrier a tile.  A row's 16-byte pieces are swizzled by a key of its
// number that spreads both the row reads (16 rows, one piece) and the transposing reads (4 rows, 64 bytes) over all banks.
//
// Bound by the matrix pipes and the vector work beside them, which add up at two waves a SIMD rather than hide each other; a third wave, and
// priorities around the products, did not help.  32/4 heads of 128, where a large library product reaches 1200 TFLOP/s: forward of one sequence of 8192
// rows 522 us, 1050 TFLOP/s; forward, dq and dk/dv of 8192 rows in 4 sequences 162, 230 and 277 us, 850, 900 and 990
// (two, three and four products); of 16384 in 11 uneven ones 347, 497 and 628, 770, 810 and 850.  Machines differ by 5 %.  Heads between the forms' sizes take
// the next one's products: 8192 rows in 4, 16/4 heads, forward us (TFLOP/s of the heads' own products) of 64 55 (620), 80 82 (520), 96 84 (620), 128 88 (780),
// 136 196 (370), 160 197 (430), 192 199 (520), 256 204 (670).
//
// Weights and ds are rounded to bf16 in front of their products, because the matrix instruction takes them so; in two pieces each they would be half as many
// products again.  Relative L2 distance from the formula in fp64 of results and gradients as they are stored (rounding the exact ones alone: 0.0016):
// one sequence of 8192 0.0021; 4 of 2048 0.0021, dq and dk 0.0024, dv 0.0023.
#include <algorithm>

#include "attention.h"

namespace mi355 {
namespace {

template <int DP>
constexpr int kWaves = DP <= 128 ? 2 : 1;  // a SIMD, by the registers that sums and operands of a wave's rows take
// ... and at most, where LDS holds no more: a schedule for a third wave's registers takes the reads ahead away (forward of 8192 rows 504 -> 544 us)
template <int DP>
constexpr int kMostWaves = DP <= 64 ? 8 : kWaves<DP>;
constexpr int kTile = 64;     // rows of the other axis a tile
constexpr int kRows = 32;     // rows a wave
constexpr uint32_t kFarOff = 1u << 30;  // an offset past every buffer: reads zeros

// (of the low four bits of r; of three for heads beyond 128, so that rows eight apart share it: their row reads meet a bank twice)
template <int DP>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  return ((r & 3) << 2) | ((r >> 2) & (DP == 128 ? 3 : 1));
}

// LDS byte offsets of a lane's reads of a tile: the swizzle is an exclusive or, and so are the steps over a row's pieces
template <int DP>
struct Reads {
  uint32_t row_, turned_;
  __device__ __forceinline__ void find(int lane, uint32_t lds0) {
    const int h = lane >> 5, r = lane & 31;
    row_ = lds0 + r * DP * 2 + ((h ^ swizzle<DP>(r)) << 4);
    const int i = lane & 15, side = (lane >> 4) & 1, t = 4 * h + (i >> 2);
    turned_ = lds0 + t * DP * 2 + (((2 * side + ((i & 3) >> 1)) ^ swizzle<DP>(t)) << 4) + 8 * (i & 1);
  }
  // the same, to be formed from here on: what is formed from these is otherwise held in registers over the loop
  __device__ __forceinline__ Reads here() const { return {static_cast<uint32_t>(opaque(row_)), static_cast<uint32_t>(opaque(turned_))}; }
  // 8 elements of row lane % 32, step kk
  __device__ __forceinline__ uint32_t row(int kk) const { return row_ ^ (kk << 5); }
  // elements 32 n + lane % 32 of rows 4 h + {0..3}, or 8 rows on
  __device__ __forceinline__ uint32_t turned(int n, int half) const { return (turned_ ^ (n << 6) ^ (DP <= 128 ? half << 5 : 0)) + half * 8 * DP * 2; }
};

__device__ __forceinline__ bf16x8 read_row(uint32_t at) { return lds_read16(at); }
template <int DP>
__device__ __forceinline__ bf16x8 read_turned(const Reads<DP>& reads, int n, uint32_t rows) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(reads.turned(n, 0) + rows));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(reads.turned(n, 1) + rows));
  const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, v);
}

// Requests of a workgroup's four waves for a tile of a head's rows, 1 KiB each: a wave's j-th brings rows of its own
template <int DP>
struct Requests {
  static constexpr int EACH = kTile * DP * 2 / 4096;  // a wave's requests a tile
  static constexpr int ROWS = 1024 / (DP * 2);        // rows a request
  uint64_t base;
  int64_t row_bytes;
  uint32_t voff;
  int end, D;
  __device__ __forceinline__ void find(const void* p, int64_t token, int end_, int D_, int lane, int wave) {
    base = reinterpret_cast<uint64_t>(p);
    row_bytes = token * 2;
    end = end_, D = D_;
    if constexpr (DP <= 128) voff = offset(lane, wave);
  }
  __device__ __forceinline__ uint32_t offset(int lane, int wave) const {
    constexpr int CPR = DP / 8;
    // (a wave's requests are 4 ROWS = 32, 16 or 8 rows apart: the same swizzle)
    const int r = ROWS * wave + lane / CPR, c = (lane % CPR) ^ swizzle<DP>(r);
    return c * 8 < D ? static_cast<uint32_t>(r * row_bytes) + c * 16 : kFarOff;
  }
  // rows [row0, row0 + 64) to LDS at `lds`; zeros for rows from `end` on
  __device__ __forceinline__ void request(int row0, uint32_t lds, int wave) const {
    const int64_t left = static_cast<int64_t>(end - 1 - row0) * row_bytes + D * 2;
    const uint32_t bytes = left < 0 ? 0 : left < kFarOff ? static_cast<uint32_t>(left) : kFarOff;
    const uint64_t at = base + static_cast<int64_t>(row0) * row_bytes;
    const uint32_t step = 4 * ROWS * static_cast<uint32_t>(row_bytes);
    uint32_t off;
    if constexpr (DP <= 128) off = opaque(voff);
    else off = offset(lane_anew(), wave);
#pragma unroll
    for (int j = 0; j < EACH; ++j) lds_load16_within(at, bytes, off + j * step, lds + (4 * j + wave) * 1024);
  }
};

// a wave's own 32 rows as right operand: 8 elements of row lane % 32 a step, zeros where `on` is not set
template <int DP>
__device__ __forceinline__ void own_rows(bf16x8 (&x)[DP / 16], const uint16_t* row, bool on, int D, int lane) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int d = 16 * kk + 8 * (lane >> 5);
    u32x4 v = {0, 0, 0, 0};
    if (on && d < D) v = *reinterpret_cast<const u32x4*>(row + d);
    x[kk] = __builtin_bit_cast(bf16x8, v);
  }
}
// Waits for the operands here: the compiler, which does not count requests to LDS, would wait in the loop, for all that are under way.
template <int N>
__device__ __forceinline__ void settle(bf16x8 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zeros() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// the value of the other lane half, both in one
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int least(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int most(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

// rows 16 kk + ... of a 32 x 32 result as the right operand of the next product
__device__ __forceinline__ bf16x8 operand_of(const f32x16& s, int kk) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(s[8 * kk + 2 * i], s[8 * kk + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, v);
}

// what rounding took from the operand above, as an operand of its own
__device__ __forceinline__ bf16x8 rest_of(const f32x16& s, int kk, const bf16x8& rounded) {
  f32x16 left;
#pragma unroll
  for (int i = 0; i < 8; ++i) left[8 * kk + i] = s[8 * kk + i] - static_cast<float>(rounded[i]);
  return operand_of(left, kk);
}

// elements 32 n + 8 (2 a + h) .. + 7 of the lane's row from a turned result's block: lane half h's pieces of 4 exchanged for whole ones of 8
__device__ __forceinline__ void eight_of(const f32x16& o, int a, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[8 * a + i]), __float_as_uint(o[8 * a + 4 + i]), false, false);
    v[i] = __uint_as_float(r[0]);
    v[4 + i] = __uint_as_float(r[1]);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
  return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

__device__ __forceinline__ void put8(uint16_t* to, const float (&v)[8]) { *reinterpret_cast<u32x4*>(to) = pack8(v); }
__device__ __forceinline__ void put8(float* to, const float (&v)[8]) {
  reinterpret_cast<f32x4*>(to)[0] = f32x4{v[0], v[1], v[2], v[3]};
  reinterpret_cast<f32x4*>(to)[1] = f32x4{v[4], v[5], v[6], v[7]};
}

// The first `rows` of the wave's 32 result rows, `D` elements each, to `to` + row * pitch; eight(n, a, v) gives elements 32 n + 16 a + 8 half ..
// + 7 of the lane's row.  Rows that are whole numbers of 16 bytes are stored from the registers.  Others, whose elements lie anywhere, pass
// through the wave's quarter of LDS (which everyone is done with by then) and go out row by row, lanes side by side: an
// element a lane of 32 rows at once took 104 us of a forward's 296 (8192 rows, 16 heads of 150).
template <int DP, typename E, typename Eight>
__device__ __forceinline__ void store_rows(E* to, int64_t pitch, int rows, int D, uint16_t* smem, int wave, int lane, Eight eight) {
  const int half = lane >> 5, row = lane & 31;
  constexpr int WHOLE = 16 / sizeof(E);
  E* part = reinterpret_cast<E*>(smem) + wave * 32 * DP;
  auto at = [&](int r, int d) { return r * DP + (((d / WHOLE) ^ (r & 7)) * WHOLE) + d % WHOLE; };
  const bool whole = D % 8 == 0;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      float v[8];
      eight(n, a, v);
      const int d = 32 * n + 16 * a + 8 * half;
      if (whole) {
        if (row < rows && d < D) put8(to + row * pitch + d, v);
      } else if constexpr (sizeof(E) == 2) {
        put8(part + at(row, d), v);
      } else {
        *reinterpret_cast<f32x4*>(part + at(row, d)) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(part + at(row, d + 4)) = f32x4{v[4], v[5], v[6], v[7]};
      }
    }
  if (whole) return;
  wave_lds_sync();
  if (sizeof(E) == 2 && D % 2 == 0) {  // two elements of 2 bytes a lane
    for (int r = 0; r < rows; ++r)
      for (int d = 2 * lane; d < D; d += 2 * kWave)
        *reinterpret_cast<uint32_t*>(to + r * pitch + d) = *reinterpret_cast<const uint32_t*>(part + at(r, d));
  } else {
    for (int r = 0; r < rows; ++r)
      for (int d = lane; d < D; d += kWave) to[r * pitch + d] = part[at(r, d)];
  }
  wave_lds_sync();  // read before the next result's rows come
}

// the workgroup's range over the other axis and the wave's, from every lane's row's
struct Ranges {
  int lo, hi, first, last;  // workgroup: [lo, hi), wave: [first, last)
  __device__ __forceinline__ void find(int lane_lo, int lane_hi, int* red, int wave) {
    first = least(lane_lo);
    last = most(lane_hi);
    if ((threadIdx.x & 63) == 0) red[2 * wave] = first, red[2 * wave + 1] = last;
    __syncthreads();
    lo = __builtin_amdgcn_readfirstlane(min(min(red[0], red[2]), min(red[4], red[6])));
    hi = __builtin_amdgcn_readfirstlane(max(max(red[1], red[3]), max(red[5], red[7])));
    __syncthreads();
  }
};

// ds in two bf16 pieces instead of one where a wave has rows (keys) of a sequence shorter than its own 32: decided by the wave, so that a sequence's
// gradients do not depend on what it is packed with.  Of sequences of 2 to 31 rows dq and dk are 1.52 to 1.47 times as far from the formula as rounding
// the exact gradients takes them with one piece, 1.15 to 1.08 with two, at heads of 64, 128 and 200 alike (relative L2); there is no length at which the error
// changes.  Such sequences lie in masked tiles only, where the second piece's products stand, so the others' code is the same with it and without: 120
// sequences in 5003 rows, 16 heads of 64, 78.5 us without, 81.2 with; 8192 rows in 4 704 either way.  Longer ones have tiles without masked places, in which a
// second piece would be a third (dq) or a quarter (dk, dv) more products.
constexpr int kShort = 32;

constexpr float kGrowth = 8.0f;  // a row's weights stay below 2^8 of its reference: the reference follows its maximum in such steps

template <int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kWaves<DP>, kMostWaves<DP>))) void bf16_forward_kernel(const AttnArgs p, int tiles) {
  constexpr int KK = DP / 16, NB = DP / 32;
  constexpr uint32_t TILE_BYTES = kTile * DP * 2;
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_cptr)smem));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const Place at = place_of(blockIdx.x, p.H << p.share_bits, tiles, p.query_order, true);
  const int h = at.head >> p.share_bits, share = at.head - (h << p.share_bits), g = h / p.group;
  const int row0 = at.tile * 4 * kRows + wave * kRows, row = row0 + (lane & 31);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, row, start, end);
  const bool on = start < end;
  Ranges range;
  range.find(on ? start : p.T, on ? row + 1 : 0, reinterpret_cast<int*>(smem), wave);
  take_share(range.lo, range.hi, kTile, share, p.share_bits);
  const int latest = most(on ? start : p.T);  // keys from here to the wave's first row are seen by all its rows
  Reads<DP> reads;
  reads.find(lane, lds0);
  Requests<DP> keys, values;
  keys.find(static_cast<const uint16_t*>(p.k) + g * p.k_head, p.k_token, range.hi, p.D, lane, wave);
  values.find(static_cast<const uint16_t*>(p.v) + g * p.v_head, p.v_token, range.hi, p.D, lane, wave);
  auto request = [&](int k0, uint32_t buffer) {
    keys.request(k0, lds0 + buffer * 2 * TILE_BYTES, wave);
    values.request(k0, lds0 + buffer * 2 * TILE_BYTES + TILE_BYTES, wave);
  };
  if (range.lo < range.hi) request(range.lo, 0);
  bf16x8 q[KK];
  own_rows<DP>(q, row_at<uint16_t>(p.q, p.q_token, p.q_head, min(row, p.T - 1), h), on, p.D, lane);
  settle(q);
  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = zeros();
  float m = kNegInf, ref = 0.0f, l = 0.0f;
  const float c = p.c, growth = kGrowth / p.c;
  auto tile = [&](int k0, auto which) {
    constexpr uint32_t BUFFER = decltype(which)::value;
    lds_wait<0>();
    lds_sync<63>();  // everyone's requests of this tile have landed, and everyone has read the other buffer
    if (k0 + kTile < range.hi) request(k0 + kTile, BUFFER ^ 1);
    if (k0 >= range.last || k0 + kTile <= range.first) return;
    constexpr uint32_t kt = BUFFER * 2 * TILE_BYTES, vt = kt + TILE_BYTES;
    f32x16 s[2] = {zeros(), zeros()};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma(read_row(reads.row(kk) + kt + b * 32 * DP * 2), q[kk], s[b]);
    reads_first<6>();
    interleave<2 * KK - 6, 1, 0>();
    interleave<6, 0, 0>();
    if (k0 + kTile - 1 > row0 || k0 < latest) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = k0 + 32 * b + 8 * (i >> 2) + 4 * half + (i & 3);
          s[b][i] = on && key >= start && key <= row ? s[b][i] : kNegInf;
        }
    }
    float top = kNegInf;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = halves_max(top);
    if (__any(top > m + growth)) {
      const float next = fmaxf(m, top), next_ref = next == kNegInf ? 0.0f : next * c;  // (nothing seen yet: weights of 0, not NaN)
      const float keep = m == kNegInf ? 0.0f : exp2_f32(ref - next_ref);
      l *= keep;
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n] *= keep;
      m = next;
      ref = next_ref;
    }
    // 16 keys a step: the matrix instructions of one beside the exponentials of the next
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 8 * (t & 1); i < 8 * (t & 1) + 8; ++i) {
        s[t >> 1][i] = exp2_f32(fmaf(s[t >> 1][i], c, -ref));
        part[i & 1] += s[t >> 1][i];
      }
      l += part[0] + part[1];
      const bf16x8 w = operand_of(s[t >> 1], t & 1);
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n] = mfma(read_turned(reads, n, vt + t * 16 * DP * 2), w, o[n]);
    }
    reads_first<2 * NB>();
    __builtin_amdgcn_sched_group_barrier(0x002, 30, 0);
    interleave<3 * NB, 2, 32 / NB>();
    interleave<NB, 0, 0>();
  };
  for (int k0 = range.lo; k0 < range.hi; k0 += 2 * kTile) {
    tile(k0, std::integral_constant<uint32_t, 0>{});
    if (k0 + kTile < range.hi) tile(k0 + kTile, std::integral_constant<uint32_t, 1>{});
  }
  l = halves_sum(l);
  const AttnArgs& z = late_arguments();
  const bool nothing = z.share_bits && l == 0.0f;  // a share without a key of the row's: nothing to add
  const float inverse = 1.0f / l, lse = !on ? INFINITY : nothing ? kNegInf : ref + log2f(l);
  bool spoilt = false;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[n][i] = on && !nothing ? o[n][i] * inverse : 0.0f;
      spoilt |= o[n][i] != o[n][i];
    }
  if (z.D_out % 8) __syncthreads();
  const int rows = min(max(z.T - row0, 0), kRows);
  const int64_t dense = (static_cast<int64_t>(row0) * z.H + h) * z.D_out, pitch = static_cast<int64_t>(z.H) * z.D_out;
  auto eight = [&](int n, int a, float (&v)[8]) __attribute__((always_inline)) { eight_of(o[n], a, v); };
  if (z.share_bits) {
    store_rows<DP>(z.out_part + static_cast<int64_t>(share) * z.T * pitch + dense, pitch, rows, z.D_out, smem, wave, lane, eight);
    if (half == 0 && row < z.T) z.lse_part[(static_cast<int64_t>(share) * z.H + h) * z.T + row] = lse;
  } else {
    store_rows<DP>(static_cast<uint16_t*>(z.out) + dense, pitch, rows, z.D_out, smem, wave, lane, eight);
    if (z.rest)
      store_rows<DP>(static_cast<uint16_t*>(z.rest) + dense, pitch, rows, z.D_out, smem, wave, lane,
                     [&](int n, int a, float (&v)[8]) __attribute__((always_inline)) {
                       eight_of(o[n], a, v);
                       const u32x4 packed = pack8(v);
#pragma unroll
                       for (int i = 0; i < 8; ++i) v[i] -= __uint_as_float(i & 1 ? packed[i / 2] & 0xffff0000u : packed[i / 2] << 16);
                     });
    if (half == 0 && z.lse && row < z.T) z.lse[static_cast<int64_t>(h) * z.T + row] = lse;
  }
  // (a sum that is NaN, or zero: every element is NaN by the row's own scores)
  const uint64_t again = __ballot(spoilt && l == l && l != 0.0f && row < z.T);
  if (!again) return;
  lds_wait<0>();
  rows_again<uint16_t, false>(z, h, row0, static_cast<uint32_t>(again | again >> 32), start, lse, 0.0f, range.lo, range.hi,
                          whole_tiles(range.lo, range.hi, kTile, latest, row0 + 1), share);
}

// dq, and delta for the kernel behind this one
template <int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kWaves<DP>, kMostWaves<DP>))) void bf16_dq_kernel(const AttnArgs p, int tiles) {
  constexpr int KK = DP / 16, NB = DP / 32;
  constexpr uint32_t TILE_BYTES = kTile * DP * 2;
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_cptr)smem));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const Place at = place_of(blockIdx.x, p.H << p.share_bits, tiles, p.query_order, true);
  const int h = at.head >> p.share_bits, share = at.head - (h << p.share_bits), g = h / p.group;
  const int row0 = at.tile * 4 * kRows + wave * kRows, row = row0 + (lane & 31);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, row, start, end);
  const bool on = start < end, several = on && start < row;  // (a row that sees one key: its weight is 1, whatever its score)
  Ranges range;
  range.find(on ? start : p.T, on ? row + 1 : 0, reinterpret_cast<int*>(smem), wave);
  take_share(range.lo, range.hi, kTile, share, p.share_bits);
  const int latest = most(on ? start : p.T);
  const bool fine = __any(on && end - start < kShort);
  Reads<DP> reads;
  reads.find(lane, lds0);
  Requests<DP> keys, values;
  keys.find(static_cast<const uint16_t*>(p.k) + g * p.k_head, p.k_token, range.hi, p.D, lane, wave);
  values.find(static_cast<const uint16_t*>(p.v) + g * p.v_head, p.v_token, range.hi, p.D, lane, wave);
  auto request = [&](int k0, uint32_t buffer) {
    keys.request(k0, lds0 + buffer * 2 * TILE_BYTES, wave);
    values.request(k0, lds0 + buffer * 2 * TILE_BYTES + TILE_BYTES, wave);
  };
  if (range.lo < range.hi) request(range.lo, 0);
  const int here = min(row, p.T - 1);
  const int64_t dense = (static_cast<int64_t>(here) * p.H + h) * p.D;
  bf16x8 q[KK], dout[KK];
  own_rows<DP>(q, row_at<uint16_t>(p.q, p.q_token, p.q_head, here, h), on, p.D, lane);
  own_rows<DP>(dout, static_cast<const uint16_t*>(p.dout) + dense, on, p.D, lane);
  float delta = 0.0f;
  {
    auto dot = [&](const void* base) {
      bf16x8 x[KK];
      own_rows<DP>(x, static_cast<const uint16_t*>(base) + dense, on, p.D, lane);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = fmaf(static_cast<float>(x[kk][i]), static_cast<float>(dout[kk][i]), delta);
    };
    dot(p.o);
    if (p.rest) dot(p.rest);
  }
  delta = halves_sum(delta);
  const float lse = on ? p.lse[static_cast<int64_t>(h) * p.T + row] : INFINITY;
  if (half == 0 && row < p.T && share == 0) {  // as the kernel behind this one starts its sums from: -lse / c and -delta
    p.delta[static_cast<int64_t>(h) * p.T + row] = on ? -delta : 0.0f;
    p.delta[static_cast<int64_t>(p.H + h) * p.T + row] = -lse / p.c;
  }
  settle(q);
  settle(dout);
  f32x16 dq[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) dq[n] = zeros();
  const float c = p.c;
  auto tile = [&](int k0, auto which) {
    constexpr uint32_t BUFFER = decltype(which)::value;
    lds_wait<0>();
    lds_sync<63>();
    if (k0 + kTile < range.hi) request(k0 + kTile, BUFFER ^ 1);
    if (k0 >= range.last || k0 + kTile <= range.first) return;
    constexpr uint32_t kt = BUFFER * 2 * TILE_BYTES, vt = kt + TILE_BYTES;
    const bool masked = k0 + kTile - 1 > row0 || k0 < latest;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 s = zeros(), ds = zeros();
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        s = mfma(read_row(reads.row(kk) + kt + b * 32 * DP * 2), q[kk], s);
        ds = mfma(read_row(reads.row(kk) + vt + b * 32 * DP * 2), dout[kk], ds);
      }
      reads_first<4>();
      interleave<2 * KK - 4, 1, 0>();
      interleave<4, 0, 0>();
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] = exp2_f32(fmaf(s[i], c, -lse)) * (ds[i] - delta);
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = k0 + 32 * b + 8 * (i >> 2) + 4 * half + (i & 3);
          ds[i] = several && key >= start && key <= row ? ds[i] : 0.0f;
        }
        if (fine) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bf16x8 left = rest_of(ds, t, operand_of(ds, t));
#pragma unroll
            for (int n = 0; n < NB; ++n) dq[n] = mfma(read_turned(reads, n, kt + (2 * b + t) * 16 * DP * 2), left, dq[n]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 w = operand_of(ds, t);
#pragma unroll
        for (int n = 0; n < NB; ++n) dq[n] = mfma(read_turned(reads, n, kt + (2 * b + t) * 16 * DP * 2), w, dq[n]);
      }
      reads_first<8>();
      interleave<2 * NB - 4, 2, 0>();
      interleave<4, 0, 0>();
    }
  };
  for (int k0 = range.lo; k0 < range.hi; k0 += 2 * kTile) {
    tile(k0, std::integral_constant<uint32_t, 0>{});
    if (k0 + kTile < range.hi) tile(k0 + kTile, std::integral_constant<uint32_t, 1>{});
  }
  const AttnArgs& z = late_arguments();
  bool spoilt = false;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dq[n][i] = on ? dq[n][i] * z.scale : 0.0f;
      spoilt |= dq[n][i] != dq[n][i];
    }
  if (z.D_out % 8) __syncthreads();
  const int rows = min(max(z.T - row0, 0), kRows);
  const int64_t dense_dq = (static_cast<int64_t>(row0) * z.H + h) * z.D_out, pitch = static_cast<int64_t>(z.H) * z.D_out;
  auto eight = [&](int n, int a, float (&v)[8]) __attribute__((always_inline)) { eight_of(dq[n], a, v); };
  if (z.share_bits)
    store_rows<DP>(z.dq_part + static_cast<int64_t>(share) * z.T * pitch + dense_dq, pitch, rows, z.D_out, smem, wave, lane, eight);
  else
    store_rows<DP>(static_cast<uint16_t*>(z.dq) + dense_dq, pitch, rows, z.D_out, smem, wave, lane, eight);
  // (NaN statistics: every element is NaN by the row's own keys; but for a row that sees one, which has no gradient at all)
  const uint64_t again = __ballot(spoilt && !(several && (lse != lse || delta != delta)) && row < z.T);
  if (!again) return;
  lds_wait<0>();
  rows_again<uint16_t, true>(z, h, row0, static_cast<uint32_t>(again | again >> 32), start, lse, delta, range.lo, range.hi,
                     whole_tiles(range.lo, range.hi, kTile, latest, row0 + 1), share);
}

// dk and dv: a wave's 32 keys against the query heads of their group, or a part of them
template <int DP>
__global__ __launch_bounds__(256, kWaves<DP>) void bf16_dkv_kernel(const AttnArgs p, int tiles) {
  constexpr int KK = DP / 16, NB = DP / 32;
  constexpr uint32_t TILE_BYTES = kTile * DP * 2, STAGE = 2 * TILE_BYTES + 512;  // queries, gradients, -lse / c, -delta
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_cptr)smem));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const Place at = place_of(blockIdx.x, p.G * p.splits, tiles, p.key_order, false);
  const int g = at.head / p.splits, split = at.head % p.splits;
  const int parts = p.splits >> p.key_share_bits, heads = (p.group + parts - 1) / parts;
  const int h0 = g * p.group + (split >> p.key_share_bits) * heads, h1 = min(h0 + heads, (g + 1) * p.group);
  const int key0 = at.tile * 4 * kRows + wave * kRows, key = key0 + (lane & 31);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, key, start, end);
  const bool on = start < end;
  // bit 0: the first row of a sequence sees this key only: its weight is 1, whatever its score; bit 1: of a short sequence
  const int alone = (key == start) | (on && end - start < kShort) << 1;
  Ranges range;
  range.find(on ? key : p.T, on ? end : 0, reinterpret_cast<int*>(smem), wave);
  take_share(range.lo, range.hi, kTile, split & ((1 << p.key_share_bits) - 1), p.key_share_bits);
  const int earliest = least(on ? end : 0);  // rows from the wave's last key to here see all its keys
  Reads<DP> reads;
  reads.find(lane, lds0);
  const int here = min(key, p.T - 1);
  bf16x8 k[KK], v[KK];
  own_rows<DP>(k, row_at<uint16_t>(p.k, p.k_token, p.k_head, here, g), on, p.D, lane);
  own_rows<DP>(v, row_at<uint16_t>(p.v, p.v_token, p.v_head, here, g), on, p.D, lane);
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) dk[n] = zeros(), dv[n] = zeros();
  const float c = p.c;
  Requests<DP> queries, grads;
  queries.find(p.q, p.q_token, range.hi, p.D, lane, wave);
  grads.find(p.dout, static_cast<int64_t>(p.H) * p.D, range.hi, p.D, lane, wave);
  const int steps = range.lo < range.hi ? (range.hi - range.lo + kTile - 1) / kTile : 0;
  auto request = [&](int h, int r0, uint32_t buffer) {
    const uint32_t to = lds0 + buffer * STAGE;
    queries.base = reinterpret_cast<uint64_t>(static_cast<const uint16_t*>(p.q) + h * p.q_head);
    grads.base = reinterpret_cast<uint64_t>(static_cast<const uint16_t*>(p.dout) + h * p.D);
    queries.request(r0, to, wave);
    grads.request(r0, to + TILE_BYTES, wave);
    if (wave < 2) {  // -lse / c and -delta of the tile's 64 rows, one wave each
      const float* from = p.delta + static_cast<int64_t>(wave ? h : p.H + h) * p.T;
      lds_load4_within(reinterpret_cast<uint64_t>(from + r0), static_cast<uint32_t>(min(p.T - r0, kTile)) * 4, lane * 4,
                       to + 2 * TILE_BYTES + wave * 256);
    }
  };
  settle(k);
  settle(v);
  auto tile = [&](int h, int t, auto which) {
    constexpr uint32_t BUFFER = decltype(which)::value;
    const int r0 = range.lo + t * kTile;
    lds_wait<0>();
    lds_sync<63>();
    if (t + 1 < steps) request(h, r0 + kTile, BUFFER ^ 1);
    else if (h + 1 < h1) request(h + 1, range.lo, BUFFER ^ 1);
    if (r0 >= range.last || r0 + kTile <= range.first) return;
    constexpr uint32_t qt = BUFFER * STAGE, dt = qt + TILE_BYTES, stats = dt + TILE_BYTES;
    const bool masked = r0 < key0 + kRows - 1 || r0 + kTile > earliest;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const Reads<DP> at_tile = reads.here();
      const uint32_t from_stats = lds0 + 16 * (lane_anew() >> 5);
      f32x16 s, ds;  // from -lse / c and -delta of the lane's rows
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 x = *lds_at<const f32x4>(from_stats + stats + (32 * b + 8 * a) * 4);
        const f32x4 y = *lds_at<const f32x4>(from_stats + stats + 256 + (32 * b + 8 * a) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * a + i] = x[i], ds[4 * a + i] = y[i];
      }
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        s = mfma(read_row(at_tile.row(kk) + qt + b * 32 * DP * 2), k[kk], s);
        ds = mfma(read_row(at_tile.row(kk) + dt + b * 32 * DP * 2), v[kk], ds);
      }
      if constexpr (DP <= 128) {  // (larger heads have no registers for reads ahead)
        reads_first<12>();
        interleave<2 * KK - 4, 1, 0>();
        interleave<4, 0, 0>();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_f32(s[i] * c);
        ds[i] *= s[i];
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = r0 + 32 * b + 8 * (i >> 2) + 4 * half + (i & 3);
          const bool seen = on && r >= key && r < end;
          s[i] = seen ? s[i] : 0.0f;
          ds[i] = seen && r >= key + (alone & 1) ? ds[i] : 0.0f;
        }
        if (__any(alone & 2)) {
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2) {
            const bf16x8 left = rest_of(ds, t2, operand_of(ds, t2));
#pragma unroll
            for (int n = 0; n < NB; ++n) dk[n] = mfma(read_turned(at_tile, n, qt + (2 * b + t2) * 16 * DP * 2), left, dk[n]);
          }
        }
      }
      bf16x8 w[4];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) w[t2] = operand_of(s, t2), w[2 + t2] = operand_of(ds, t2);
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int n = 0; n < NB; ++n) dv[n] = mfma(read_turned(at_tile, n, dt + (2 * b + t2) * 16 * DP * 2), w[t2], dv[n]);
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int n = 0; n < NB; ++n) dk[n] = mfma(read_turned(at_tile, n, qt + (2 * b + t2) * 16 * DP * 2), w[2 + t2], dk[n]);
      if constexpr (DP <= 128) {
        reads_first<8>();
        interleave<4 * NB - 4, 2, 0>();
        interleave<4, 0, 0>();
      }
    }
  };
  if (steps) request(h0, range.lo, 0);
  const int all = steps * max(h1 - h0, 0);  // tiles, the first head's first
  for (int n = 0, h = h0, t = 0; n < all; n += 2) {
    tile(h, t, std::integral_constant<uint32_t, 0>{});
    if (++t == steps) t = 0, ++h;
    if (n + 1 == all) break;
    tile(h, t, std::integral_constant<uint32_t, 1>{});
    if (++t == steps) t = 0, ++h;
  }
  const AttnArgs& z = late_arguments();
  bool spoilt = false;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dk[n][i] = on ? dk[n][i] * z.scale : 0.0f;
      dv[n][i] = on ? dv[n][i] : 0.0f;
      spoilt |= dk[n][i] != dk[n][i] || dv[n][i] != dv[n][i];
    }
  if (z.D_out % 8) __syncthreads();
  const int lane_now = lane_anew();
  const int rows = min(max(z.T - key0, 0), kRows);
  const int64_t dense = (static_cast<int64_t>(key0) * z.G + g) * z.D_out, pitch = static_cast<int64_t>(z.G) * z.D_out;
  auto store = [&](void* to, float* parts, const f32x16 (&x)[NB]) __attribute__((always_inline)) {
    auto eight = [&](int n, int a, float (&v)[8]) __attribute__((always_inline)) { eight_of(x[n], a, v); };
    if (z.splits > 1)
      store_rows<DP>(parts + static_cast<int64_t>(split) * z.T * z.G * z.D_out + dense, pitch, rows, z.D_out, smem, wave, lane_now, eight);
    else
      store_rows<DP>(static_cast<uint16_t*>(to) + dense, pitch, rows, z.D_out, smem, wave, lane_now, eight);
  };
  store(z.dk, z.dk_part, dk);
  store(z.dv, z.dv_part, dv);
  const uint64_t again = __ballot(spoilt && key0 + (lane_now & 31) < z.T);
  if (!again) return;
  lds_wait<0>();
  int first, last;
  sequence_of(z.cu, z.sequences, z.T, key0 + (lane_now & 31), first, last);
  keys_again<uint16_t>(z, g, key0, static_cast<uint32_t>(again | again >> 32), first, last, h0, h1, range.lo, range.hi,
                      whole_tiles(range.lo, range.hi, kTile, key0 + kRows - 1, earliest), split, -1.0f);
}

template <int DP>
constexpr uint32_t kForwardLds = 4 * kTile * DP * 2;
template <int DP>
constexpr uint32_t kDkvLds = 4 * kTile * DP * 2 + 1024;

template <typename K>
void allow(K kernel, size_t bytes, PerDeviceOnce& once) {
  if (bytes <= 65536 || !once.needed()) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  once.done();
}

template <int DP>
void forward(const AttnArgs& p, hipStream_t s) {
  static PerDeviceOnce once;
  allow(bf16_forward_kernel<DP>, kForwardLds<DP>, once);
  const int tiles = (p.T + 4 * kRows - 1) / (4 * kRows);
  hipLaunchKernelGGL(bf16_forward_kernel<DP>, dim3((tiles * p.H) << p.share_bits), dim3(256), kForwardLds<DP>, s, p, tiles);
}

template <int DP>
void backward(const AttnArgs& p, hipStream_t s) {
  static PerDeviceOnce once_q, once_kv;
  allow(bf16_dq_kernel<DP>, kForwardLds<DP>, once_q);
  allow(bf16_dkv_kernel<DP>, kDkvLds<DP>, once_kv);
  const int tiles = (p.T + 4 * kRows - 1) / (4 * kRows);
  hipLaunchKernelGGL(bf16_dq_kernel<DP>, dim3((tiles * p.H) << p.share_bits), dim3(256), kForwardLds<DP>, s, p, tiles);
  hipLaunchKernelGGL(bf16_dkv_kernel<DP>, dim3(tiles * p.G * p.splits), dim3(256), kDkvLds<DP>, s, p, tiles);
}

}  // namespace

bool attention_bf16_covers(const AttnArgs& p) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                   reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.dout);
  if (p.o) bits |= reinterpret_cast<uintptr_t>(p.rest);
  if (p.D_out % 8 == 0)  // (else results go out element by element)
    bits |= reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.rest) | reinterpret_cast<uintptr_t>(p.dq) |
            reinterpret_cast<uintptr_t>(p.dk) | reinterpret_cast<uintptr_t>(p.dv);
  const int64_t sizes = p.D | p.q_token | p.q_head | p.k_token | p.k_head | p.v_token | p.v_head;
  // a tile's rows lie within 32-bit offsets of its first one
  const int64_t reach = std::max(std::max(p.q_token, p.k_token), std::max<int64_t>(p.v_token, static_cast<int64_t>(p.H) * p.D));
  return bits % 16 == 0 && sizes % 8 == 0 && reach < (1 << 22);
}

int attention_bf16_rows() { return 4 * kRows; }

void attention_bf16_forward(const AttnArgs& p, hipStream_t s) {
  if (p.D <= 64) forward<64>(p, s);
  else if (p.D <= 128) forward<128>(p, s);
  else forward<256>(p, s);
}

void attention_bf16_backward(const AttnArgs& p, hipStream_t s) {
  if (p.D <= 64) backward<64>(p, s);
  else if (p.D <= 128) backward<128>(p, s);
  else backward<256>(p, s);
}

}  // namespace mi355
