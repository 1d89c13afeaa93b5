// Causal attention over packed sequences (attention.h has the formulas) in fp32, for every head size up to 256, on
// v_mfma_f32_16x16x4_f32: fp32 products throughout.  And the entry points of both types, the order of the tiles, and what joins parts.
//
// v_mfma_f32_16x16x4_f32 takes one element a lane of each operand (row or column lane % 16, k = lane / 16) and yields four
// (column lane % 16, rows 4 (lane / 16) + i).  Products are formed turned so that one's result is the next one's operand as it lies:
//   forward, dq:  s^T = K Q^T (columns: the wave's 16 queries) is the right operand of o^T += V^T p^T and dq^T += K^T ds^T,
//   dk, dv:       s = Q K^T (columns: the wave's 16 keys) that of dv^T += dO^T p and dk^T += Q^T ds.
// Keys 4 g + i of a block then meet in step i from lane group g; the contraction over a head's elements takes them in the order
// 4 g + i of each 16 too, so that a lane reads 16 bytes of a row for four steps.
//
// Rows of the other operand pass through LDS in tiles of 32 a wave column, at a pitch of 4 floats beyond the head: the row reads
// (16 rows, 16 bytes) and the column reads (four rows 4 apart, 16 floats) both meet every bank once.  The next tile is on its way to registers
// while this one is read.
//
// A workgroup is four waves: two groups of 16 rows by two parts of the other axis, each with its own running maximum and sum, joined
// through LDS at the end; four groups and one part for heads beyond 128, whose tiles would take too many registers.  Four parts of one group, and
// one of four, were no faster for heads of 64 either.
//
// Measured: 2048 rows in 3 uneven sequences, 8/2 heads of 64: forward 46 us, dq 52, dk/dv 64, where the seven products of the formulas (5.8 GFLOP) take
// 43 at the rate of a large fp32 product (137 TFLOP/s) and the kernels form nine.  512 workgroups are two waves a SIMD, and the last rows
// of a sequence see dozens of times what its first ones do.  The matrix pipes are busy a third of the time that a CU is: a wave waits as long for its turn
// to issue as for LDS, memory and barriers.  Masks only where a tile has any and offsets formed once took a ninth off the backward; backward tiles
// are dealt over two workgroups each here (share_bits).
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace mi355 {
namespace {

constexpr uint32_t kFar = 1u << 30;  // an offset past every buffer: reads zeros

__device__ __forceinline__ float4 four_at(const float* p, int n, bool vec) {  // the first n of p[0..3], zeros behind them
  if (vec) return *reinterpret_cast<const float4*>(p);
  float4 v = make_float4(0, 0, 0, 0);
  if (n > 0) v.x = p[0];
  if (n > 1) v.y = p[1];
  if (n > 2) v.z = p[2];
  if (n > 3) v.w = p[3];
  return v;
}

// Rows [row0, row0 + ROWS) of a head on their way to LDS as fp32, zeros from row `end` on and behind the head's elements: held in registers from
// where they are fetched, a tile ahead, to where the tile before has been read
template <int DP, int ROWS>
struct Staged {
  static constexpr int P = DP + 4, QUADS = DP / 4, EACH = ROWS * QUADS / 256;
  static_assert(ROWS * QUADS % 256 == 0, "whole rounds of the workgroup");
  float4 x[EACH];
  __device__ __forceinline__ void fetch(const float* base, int64_t token, int row0, int end, int D, bool vec) {
    if (vec) {  // from a buffer that ends with the last row: zeros behind it, and no branch a request
      const int64_t left = (static_cast<int64_t>(end - 1 - row0) * token + D) * sizeof(float);
      const uint32_t bytes = left < 0 ? 0 : left < kFar ? static_cast<uint32_t>(left) : kFar;
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base) + static_cast<int64_t>(row0) * token, 0, bytes, 0x00020000);
      auto offset = [&](int i) {
        const uint32_t d = (i % QUADS) * 4, at = (static_cast<uint32_t>(i / QUADS) * static_cast<uint32_t>(token) + d) * sizeof(float);
        return at | (d < static_cast<uint32_t>(D) ? 0u : kFar);  // (a tile's offsets stay below kFar)
      };
      const uint32_t first = offset(threadIdx.x);
#pragma unroll
      for (int n = 0; n < EACH; ++n) {
        // where a round of the workgroup is whole rows, the next one is as far on for every lane
        const uint32_t at = 256 % QUADS == 0 ? first + n * (256 / QUADS) * sizeof(float) * static_cast<uint32_t>(token) : offset(threadIdx.x + 256 * n);
        x[n] = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int i = threadIdx.x + 256 * n, r = row0 + i / QUADS, d = (i % QUADS) * 4;
      x[n] = make_float4(0, 0, 0, 0);
      if (r < end && d < D) x[n] = four_at(base + static_cast<int64_t>(r) * token + d, D - d, false);
    }
  }
  __device__ __forceinline__ void put(float* tile) const {
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int i = threadIdx.x + 256 * n;
      *reinterpret_cast<float4*>(tile + (i / QUADS) * P + (i % QUADS) * 4) = x[n];
    }
  }
};

// a wave's 16 rows as an operand over the head's elements: lane's row lane % 16, elements 16 j + 4 (lane / 16) + i
template <int DP>
__device__ __forceinline__ void own_rows(float (&x)[DP / 4], const float* base, int64_t token, int row, bool on, int D, bool vec, int lane) {
#pragma unroll
  for (int j = 0; j < DP / 16; ++j) {
    const int d = 16 * j + 4 * (lane >> 4);
    float4 v = make_float4(0, 0, 0, 0);
    if (on && d < D) v = four_at(base + static_cast<int64_t>(row) * token + d, D - d, vec && d + 4 <= D);
    x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
  }
}

// 16 rows of a tile times the wave's own rows, over the head's elements
template <int DP>
__device__ __forceinline__ f32x4 rows_product(const float* tile, const float (&x)[DP / 4], int lane) {
  constexpr int P = DP + 4;
  f32x4 s = {0, 0, 0, 0};
  const float* a = tile + (lane & 15) * P + 4 * (lane >> 4);
#pragma unroll
  for (int j = 0; j < DP / 16; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(a + 16 * j);
    s = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x, x[4 * j], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_16x16x4f32(v.y, x[4 * j + 1], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_16x16x4f32(v.z, x[4 * j + 2], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_16x16x4f32(v.w, x[4 * j + 3], s, 0, 0, 0);
  }
  // two reads of 16 bytes ahead of the matrix instructions
  reads_first<2>();
#pragma unroll
  for (int j = 0; j < DP / 16 - 2; ++j) {
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    reads_first<1>();
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
  return s;
}

// acc^T (head's elements x the wave's 16) += tile^T w, over 16 rows of a tile
template <int DP>
__device__ __forceinline__ void columns_product(f32x4 (&acc)[DP / 16], const float* tile, const f32x4& w, int lane) {
  constexpr int P = DP + 4;
  const float* a = tile + 4 * (lane >> 4) * P + (lane & 15);
#pragma unroll
  for (int n = 0; n < DP / 16; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i * P + 16 * n], w[i], acc[n], 0, 0, 0);
  if constexpr (DP <= 192) {  // (larger heads have no registers for it)
    reads_first<6>();  // (of 4 bytes a lane)
    interleave<DP / 4 - 6, 1, 0>();
    interleave<6, 0, 0>();
  }
}

// over the four lane groups that hold a column
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

template <int DP>
constexpr int kAnyWaves = DP <= 64 ? 3 : 1;  // of forward and dq a SIMD, at least

constexpr int kStep = 32;  // rows of the other axis that a wave takes at a time

template <int DP, int KW>
constexpr size_t kAnyLds = sizeof(float) * (KW * kStep * 2 * (DP + 4) + 128);

// the range of the workgroup from those of its waves
__device__ __forceinline__ Span group_range(int lo, int hi, int* red) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[2 * wave] = lo, red[2 * wave + 1] = hi;
  __syncthreads();
  Span r = {min(min(red[0], red[2]), min(red[4], red[6])), max(max(red[1], red[3]), max(red[5], red[7]))};
  __syncthreads();
  r.lo = __builtin_amdgcn_readfirstlane(r.lo);
  r.hi = __builtin_amdgcn_readfirstlane(r.hi);
  return r;
}

// One workgroup: the work of every tile, then a counting sort into 256 classes of it, the largest first.  Tiles of a class come in
// whatever order the counters give: it decides who starts when, not what is added to what.
__global__ __launch_bounds__(1024) void sort_tiles_kernel(const AttnArgs p, int rows, int tiles, int32_t* query_order, int32_t* key_order) {
  __shared__ int count[256], red[16], most;
  int32_t* order = blockIdx.x ? key_order : query_order;
  if (!order) return;
  auto work = [&](int tile) {
    const int first = tile * rows, last = min(first + rows, p.T) - 1;
    int start, end, start2, end2;
    sequence_of(p.cu, p.sequences, p.T, first, start, end);
    sequence_of(p.cu, p.sequences, p.T, last, start2, end2);
    if (blockIdx.x) return max(end2, last + 1) - first;
    return last + 1 - (start < end ? start : first);
  };
  int top = 1;
  for (int t = threadIdx.x; t < tiles; t += 1024) top = max(top, work(t));
  top = wave_max_i(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  if (threadIdx.x < 256) count[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) top = max(top, red[i]);
    most = top;
  }
  __syncthreads();
  const float per = 255.0f / static_cast<float>(most);
  auto class_of = [&](int tile) { return 255 - min(255, static_cast<int>(static_cast<float>(work(tile)) * per)); };
  for (int t = threadIdx.x; t < tiles; t += 1024) atomicAdd(&count[class_of(t)], 1);
  __syncthreads();
  if (threadIdx.x < 64) {  // where each class begins: four classes a lane
    int sum = 0, mine[4];
    for (int i = 0; i < 4; ++i) mine[i] = count[4 * threadIdx.x + i], sum += mine[i];
    int at = wave_scan(sum) - sum;
    for (int i = 0; i < 4; ++i) count[4 * threadIdx.x + i] = at, at += mine[i];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < tiles; t += 1024) order[atomicAdd(&count[class_of(t)], 1)] = t;
}

template <int DP, int KW>
__global__ __launch_bounds__(256, kAnyWaves<DP>) void any_forward_kernel(const AttnArgs p, int tiles, int vec) {
  constexpr int QW = 4 / KW, P = DP + 4, NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float *kt = lds, *vt = lds + KW * kStep * P, *stats = lds + 2 * KW * kStep * P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(blockIdx.x, p.H << p.share_bits, tiles, p.query_order, true);
  const int qw = wave / KW, kw = wave % KW, h = at.head >> p.share_bits, share = at.head - (h << p.share_bits), g = h / p.group;
  const int row0 = at.tile * 16 * QW, row = row0 + 16 * qw + (lane & 15);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, row, start, end);
  const bool on = start < end;
  const int lo = wave_min_i(on ? start : p.T), hi = wave_max_i(on ? row + 1 : 0);
  const int latest = wave_max_i(on ? start : p.T), first_row = row0 + 16 * qw;  // keys between them are seen by all the wave's rows
  Span all = group_range(lo, hi, reinterpret_cast<int*>(stats));
  take_share(all.lo, all.hi, KW * kStep, share, p.share_bits);
  float q[DP / 4];
  own_rows<DP>(q, static_cast<const float*>(p.q) + h * p.q_head, p.q_token, row, on, p.D, vec, lane);
  f32x4 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x4{0, 0, 0, 0};
  float m = kNegInf, ref = 0.0f, l = 0.0f;
  const float growth = 8.0f / p.c;
  Staged<DP, KW * kStep> keys, values;
  auto fetch = [&](int k0) {
    keys.fetch(static_cast<const float*>(p.k) + g * p.k_head, p.k_token, k0, all.hi, p.D, vec);
    values.fetch(static_cast<const float*>(p.v) + g * p.v_head, p.v_token, k0, all.hi, p.D, vec);
  };
  if (all.lo < all.hi) fetch(all.lo);
  for (int k0 = all.lo; k0 < all.hi; k0 += KW * kStep) {
    __syncthreads();
    keys.put(kt);
    values.put(vt);
    phase_barrier();  // (the next tile's loads stay under way across it)
    if (k0 + KW * kStep < all.hi) fetch(k0 + KW * kStep);
    const int kb = k0 + kw * kStep;
    if (kb >= hi || kb + kStep <= lo) continue;
    f32x4 s[2];
    float top = kNegInf;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = rows_product<DP>(kt + (kw * kStep + 16 * b) * P, q, lane);
      if (kb + kStep - 1 > first_row || kb < latest) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kb + 16 * b + 4 * (lane >> 4) + i;
          s[b][i] = on && key >= start && key <= row ? s[b][i] : kNegInf;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[b][i]);
    }
    top = column_max(top);
    if (__any(!(top <= m + growth))) {  // the reference follows the maximum in steps of 2^8
      const float next = fmaxf(m, top), next_ref = next == kNegInf ? 0.0f : next * p.c;  // (nothing seen yet: every weight is 0, not NaN)
      const float keep = m == kNegInf ? 0.0f : exp2_f32(ref - next_ref);
      l *= keep;
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n] *= keep;
      m = next;
      ref = next_ref;
    }
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[b][i] = exp2_f32(fmaf(s[b][i], p.c, -ref));
        sum += s[b][i];
      }
    l += sum;  // the lane group's share; the four are added at the end
    columns_product<DP>(o, vt + (kw * kStep) * P, s[0], lane);
    columns_product<DP>(o, vt + (kw * kStep + 16) * P, s[1], lane);
  }
  l = column_sum(l);
  const AttnArgs& z = late_arguments();
  // join the parts: [wave][16 rows][DP] of sums, [wave][16] of maxima and sums
  __syncthreads();
  float *sums = lds, *tops = stats, *lens = stats + 64;
  static_assert(64 * (DP + 4) <= 2 * KW * kStep * P, "the waves' sums fit in the tiles");
#pragma unroll
  for (int n = 0; n < NB; ++n)
    *reinterpret_cast<f32x4*>(sums + (wave * 16 + (lane & 15)) * P + 16 * n + 4 * (lane >> 4)) = o[n];
  if (lane < 16) tops[wave * 16 + lane] = m, lens[wave * 16 + lane] = l;
  __syncthreads();
  // a wave writes the rows that it and its parts share: 16 / KW of them
  uint32_t again = 0;
  float row_lse = 0.0f;  // lane i: of row i of the 16
  for (int i = 0; i < 16 / KW; ++i) {
    const int mine = kw * (16 / KW) + i, r = row0 + 16 * qw + mine;
    if (r >= z.T) break;
    const int first = __builtin_amdgcn_readlane(start, mine), last = __builtin_amdgcn_readlane(end, mine);
    float w[KW], best = kNegInf, len = 0.0f;
#pragma unroll
    for (int part = 0; part < KW; ++part) best = fmaxf(best, tops[(qw * KW + part) * 16 + mine]);
    const float ref = best == kNegInf ? 0.0f : best * z.c;
#pragma unroll
    for (int part = 0; part < KW; ++part) {
      const float t = tops[(qw * KW + part) * 16 + mine];
      w[part] = t == kNegInf ? 0.0f : exp2_f32(t * z.c - ref);
      len += w[part] * lens[(qw * KW + part) * 16 + mine];
      // a part without a finite score: 0 as above, unless its own sum is NaN already
      if (t == kNegInf && lens[(qw * KW + part) * 16 + mine] != 0.0f) len = NAN;
    }
    bool spoilt = false;
    const int64_t dense = (static_cast<int64_t>(r) * z.H + h) * z.D;
    const bool nothing = z.share_bits && len == 0.0f;  // a share without a key of the row's
    for (int d = lane; d < z.D; d += kWave) {
      float v = 0.0f;
#pragma unroll
      for (int part = 0; part < KW; ++part) v += w[part] * sums[((qw * KW + part) * 16 + mine) * P + d];
      v = nothing ? 0.0f : v / len;
      spoilt |= v != v;
      if (z.share_bits) z.out_part[static_cast<int64_t>(share) * z.T * z.H * z.D + dense + d] = first < last ? v : 0.0f;
      else store_result<float>(z, dense + d, first < last ? v : 0.0f);
    }
    const float lse = first >= last ? INFINITY : nothing ? kNegInf : ref + log2f(len);
    if (lane == 0 && z.share_bits) z.lse_part[(static_cast<int64_t>(share) * z.H + h) * z.T + r] = lse;
    if (lane == 0 && !z.share_bits && z.lse) z.lse[static_cast<int64_t>(h) * z.T + r] = lse;
    // (a sum that is NaN, or zero: every element is NaN by the row's own scores)
    if (first < last && len == len && len != 0.0f && __any(spoilt)) again |= 1u << mine, row_lse = lane == mine ? lse : row_lse;
  }
  if (again)
    rows_again<float, false>(z, h, row0 + 16 * qw, again, start, row_lse, 0.0f, all.lo, all.hi,
                         whole_tiles(all.lo, all.hi, kStep, latest, first_row + 1), share);
}

// dq, and delta for the kernel behind this one
template <int DP, int KW>
__global__ __launch_bounds__(256, kAnyWaves<DP>) void any_dq_kernel(const AttnArgs p, int tiles, int vec) {
  constexpr int QW = 4 / KW, P = DP + 4, NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float *kt = lds, *vt = lds + KW * kStep * P, *stats = lds + 2 * KW * kStep * P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(blockIdx.x, p.H << p.share_bits, tiles, p.query_order, true);
  const int qw = wave / KW, kw = wave % KW, h = at.head >> p.share_bits, share = at.head - (h << p.share_bits), g = h / p.group;
  const int row0 = at.tile * 16 * QW, row = row0 + 16 * qw + (lane & 15);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, row, start, end);
  const bool on = start < end;
  const int lo = wave_min_i(on ? start : p.T), hi = wave_max_i(on ? row + 1 : 0);
  const int latest = wave_max_i(on ? start : p.T), first_row = row0 + 16 * qw;  // keys between them are seen by all the wave's rows
  Span all = group_range(lo, hi, reinterpret_cast<int*>(stats));
  take_share(all.lo, all.hi, KW * kStep, share, p.share_bits);
  float q[DP / 4], dout[DP / 4];
  const int64_t dense = static_cast<int64_t>(p.H) * p.D;
  own_rows<DP>(q, static_cast<const float*>(p.q) + h * p.q_head, p.q_token, row, on, p.D, vec, lane);
  own_rows<DP>(dout, static_cast<const float*>(p.dout) + h * p.D, dense, row, on, p.D, vec, lane);
  float delta = 0.0f;
  {
    float o[DP / 4];
    own_rows<DP>(o, static_cast<const float*>(p.o) + h * p.D, dense, row, on, p.D, vec, lane);
#pragma unroll
    for (int i = 0; i < DP / 4; ++i) delta = fmaf(o[i], dout[i], delta);
  }
  delta = column_sum(delta);
  const float lse = on ? p.lse[static_cast<int64_t>(h) * p.T + row] : INFINITY;
  if (kw == 0 && lane < 16 && row < p.T && share == 0) p.delta[static_cast<int64_t>(h) * p.T + row] = on ? delta : 0.0f;
  f32x4 dq[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) dq[n] = f32x4{0, 0, 0, 0};
  Staged<DP, KW * kStep> keys, values;
  auto fetch = [&](int k0) {
    keys.fetch(static_cast<const float*>(p.k) + g * p.k_head, p.k_token, k0, all.hi, p.D, vec);
    values.fetch(static_cast<const float*>(p.v) + g * p.v_head, p.v_token, k0, all.hi, p.D, vec);
  };
  if (all.lo < all.hi) fetch(all.lo);
  for (int k0 = all.lo; k0 < all.hi; k0 += KW * kStep) {
    __syncthreads();
    keys.put(kt);
    values.put(vt);
    phase_barrier();  // (the next tile's loads stay under way across it)
    if (k0 + KW * kStep < all.hi) fetch(k0 + KW * kStep);
    const int kb = k0 + kw * kStep;
    if (kb >= hi || kb + kStep <= lo) continue;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float* kb_t = kt + (kw * kStep + 16 * b) * P;
      const f32x4 s = rows_product<DP>(kb_t, q, lane);
      const f32x4 dp = rows_product<DP>(vt + (kw * kStep + 16 * b) * P, dout, lane);
      f32x4 ds;
#pragma unroll
      for (int i = 0; i < 4; ++i) ds[i] = exp2_f32(fmaf(s[i], p.c, -lse)) * (dp[i] - delta);
      if (kb + kStep - 1 > first_row || kb < latest) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kb + 16 * b + 4 * (lane >> 4) + i;
          const bool seen = on && key >= start && key <= row && start < row;  // (a row's only weight is 1, whatever its score)
          ds[i] = seen ? ds[i] : 0.0f;
        }
      }
      columns_product<DP>(dq, kb_t, ds, lane);
    }
  }
  const AttnArgs& z = late_arguments();
  __syncthreads();
  float *sums = lds, *lses = stats, *deltas = stats + 64;
#pragma unroll
  for (int n = 0; n < NB; ++n)
    *reinterpret_cast<f32x4*>(sums + (wave * 16 + (lane & 15)) * P + 16 * n + 4 * (lane >> 4)) = dq[n];
  if (lane < 16) lses[wave * 16 + lane] = lse, deltas[wave * 16 + lane] = delta;
  __syncthreads();
  uint32_t again = 0;
  for (int i = 0; i < 16 / KW; ++i) {
    const int mine = kw * (16 / KW) + i, r = row0 + 16 * qw + mine;
    if (r >= z.T) break;
    const int first = __builtin_amdgcn_readlane(start, mine), last = __builtin_amdgcn_readlane(end, mine);
    bool spoilt = false;
    float* out = (z.share_bits ? z.dq_part + static_cast<int64_t>(share) * z.T * z.H * z.D : static_cast<float*>(z.dq)) +
                 (static_cast<int64_t>(r) * z.H + h) * z.D;
    for (int d = lane; d < z.D; d += kWave) {
      float v = 0.0f;
#pragma unroll
      for (int part = 0; part < KW; ++part) v += sums[((qw * KW + part) * 16 + mine) * P + d];
      spoilt |= v != v;
      store_from_f32<float>(out + d, first < last ? v * z.scale : 0.0f);
    }
    // (NaN statistics: every element is NaN by the row's own keys; but for a row that sees one, which has no gradient at all)
    const float row_lse = lses[(qw * KW) * 16 + mine], row_delta = deltas[(qw * KW) * 16 + mine];
    const bool own = first < r && (row_lse != row_lse || row_delta != row_delta);
    if (first < last && !own && __any(spoilt)) again |= 1u << mine;
  }
  if (again)
    rows_again<float, true>(z, h, row0 + 16 * qw, again, start, lse, delta, all.lo, all.hi, whole_tiles(all.lo, all.hi, kStep, latest, first_row + 1), share);
}

// dk and dv: a wave's 16 keys against the query heads of their group, or a part of them
template <int DP, int KW>
__global__ __launch_bounds__(256) void any_dkv_kernel(const AttnArgs p, int tiles, int vec) {
  constexpr int QW = 4 / KW, P = DP + 4, NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float *qt = lds, *dt = lds + KW * kStep * P, *stats = lds + 2 * KW * kStep * P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qw = wave / KW, kw = wave % KW;
  const Place at = place_of(blockIdx.x, p.G * p.splits, tiles, p.key_order, false);
  const int g = at.head / p.splits, split = at.head % p.splits;
  const int parts = p.splits >> p.key_share_bits, heads = (p.group + parts - 1) / parts;
  const int h0 = g * p.group + (split >> p.key_share_bits) * heads, h1 = min(h0 + heads, (g + 1) * p.group);
  const int key0 = at.tile * 16 * QW, key = key0 + 16 * qw + (lane & 15);
  int start, end;
  sequence_of(p.cu, p.sequences, p.T, key, start, end);
  const bool on = start < end;
  const int lo = wave_min_i(on ? key : p.T), hi = wave_max_i(on ? end : 0);
  const int earliest = wave_min_i(on ? end : 0), last_key = key0 + 16 * qw + 15;  // rows between them see all the wave's keys
  Span all = group_range(lo, hi, reinterpret_cast<int*>(stats));
  take_share(all.lo, all.hi, KW * kStep, split & ((1 << p.key_share_bits) - 1), p.key_share_bits);
  float k[DP / 4], v[DP / 4];
  own_rows<DP>(k, static_cast<const float*>(p.k) + g * p.k_head, p.k_token, key, on, p.D, vec, lane);
  own_rows<DP>(v, static_cast<const float*>(p.v) + g * p.v_head, p.v_token, key, on, p.D, vec, lane);
  f32x4 dk[NB], dv[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) dk[n] = dv[n] = f32x4{0, 0, 0, 0};
  const int64_t dense = static_cast<int64_t>(p.H) * p.D;
  Staged<DP, KW * kStep> queries, grads;
  auto fetch = [&](int h, int r0) {
    queries.fetch(static_cast<const float*>(p.q) + h * p.q_head, p.q_token, r0, all.hi, p.D, vec);
    grads.fetch(static_cast<const float*>(p.dout) + h * p.D, dense, r0, all.hi, p.D, vec);
  };
  if (all.lo < all.hi && h0 < h1) fetch(h0, all.lo);
  for (int h = h0; h < h1; ++h) {
    const float *lse = p.lse + static_cast<int64_t>(h) * p.T, *delta = p.delta + static_cast<int64_t>(h) * p.T;
    for (int r0 = all.lo; r0 < all.hi; r0 += KW * kStep) {
      __syncthreads();
      queries.put(qt);
      grads.put(dt);
      phase_barrier();
      if (r0 + KW * kStep < all.hi) fetch(h, r0 + KW * kStep);
      else if (h + 1 < h1) fetch(h + 1, all.lo);
      const int rb = r0 + kw * kStep;
      if (rb >= hi || rb + kStep <= lo) continue;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float *q_t = qt + (kw * kStep + 16 * b) * P, *d_t = dt + (kw * kStep + 16 * b) * P;
        const f32x4 s = rows_product<DP>(q_t, k, lane);
        const f32x4 dp = rows_product<DP>(d_t, v, lane);
        f32x4 w, ds;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = min(rb + 16 * b + 4 * (lane >> 4) + i, p.T - 1);
          w[i] = exp2_f32(fmaf(s[i], p.c, -lse[r]));
          ds[i] = w[i] * (dp[i] - delta[r]);
        }
        if (rb <= last_key || rb + kStep > earliest) {  // (the row of the key itself is masked too: a row's only weight is 1, whatever its score)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = rb + 16 * b + 4 * (lane >> 4) + i;
            const bool seen = on && r >= key && r < end;
            w[i] = seen ? w[i] : 0.0f;
            ds[i] = seen && start < r ? ds[i] : 0.0f;
          }
        }
        columns_product<DP>(dv, d_t, w, lane);
        columns_product<DP>(dk, q_t, ds, lane);
      }
    }
  }
  const AttnArgs& z = late_arguments();
  const int64_t part0 = static_cast<int64_t>(split) * z.T * z.G * z.D;
  bool spoilt[16 / KW];
#pragma unroll
  for (int i = 0; i < 16 / KW; ++i) spoilt[i] = false;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n)
      *reinterpret_cast<f32x4*>(lds + (wave * 16 + (lane & 15)) * P + 16 * n + 4 * (lane >> 4)) = which ? dk[n] : dv[n];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16 / KW; ++i) {
      const int mine = kw * (16 / KW) + i, r = key0 + 16 * qw + mine;
      if (r >= z.T) continue;
      const int first = __builtin_amdgcn_readlane(start, mine), last = __builtin_amdgcn_readlane(end, mine);
      const int64_t at = (static_cast<int64_t>(r) * z.G + g) * z.D;
      bool bad = false;
      for (int d = lane; d < z.D; d += kWave) {
        float x = 0.0f;
#pragma unroll
        for (int part = 0; part < KW; ++part) x += lds[((qw * KW + part) * 16 + mine) * P + d];
        bad |= x != x;
        x = first < last ? (which ? x * z.scale : x) : 0.0f;
        if (z.splits > 1) (which ? z.dk_part : z.dv_part)[part0 + at + d] = x;
        else store_from_f32<float>(static_cast<float*>(which ? z.dk : z.dv) + at + d, x);
      }
      spoilt[i] |= first < last && __any(bad);
    }
  }
  uint32_t again = 0;
#pragma unroll
  for (int i = 0; i < 16 / KW; ++i)
    if (spoilt[i]) again |= 1u << (kw * (16 / KW) + i);
  if (again)
    keys_again<float>(z, g, key0 + 16 * qw, again, start, end, h0, h1, all.lo, all.hi, whole_tiles(all.lo, all.hi, kStep, last_key + 1, earliest), split,
                     1.0f);
}

// bf16 heads of a size that is no whole number of 16 bytes, copied for the matrix kernels into rows that are: a wave a head, zeros behind its
// elements.  8192 rows in 4 sequences of 16/4 heads of 75, forward 113 us, forward and backward 467; in fp32 products from where they lay 1054 and 4631,
// and of 64 rows no faster.
struct PadArgs {
  const uint16_t* from[6];
  uint16_t* to[6];
  int64_t token[6], head[6];
  int heads[6];
  int D, D8;
  int64_t T;
};
constexpr int kPadRows = 8;  // heads a wave: their loads are under way together
__global__ __launch_bounds__(256) void pad_heads_kernel(const PadArgs p) {
  typedef uint32_t __attribute__((aligned(2))) two;  // two elements, wherever they begin
  const int n = blockIdx.y, lane = threadIdx.x & 63;
  const uint32_t heads = p.heads[n], rows = static_cast<uint32_t>(p.T) * heads;
  // (T x heads is under 2^31)
  for (uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kPadRows; first < rows; first += gridDim.x * 4 * kPadRows) {
    const uint16_t* from[kPadRows];
#pragma unroll
    for (int i = 0; i < kPadRows; ++i) {
      const uint32_t row = min(first + i, rows - 1), t = row / heads, h = row - t * heads;
      from[i] = p.from[n] + t * p.token[n] + h * p.head[n];
    }
    uint16_t* to = p.to[n] + static_cast<int64_t>(first) * p.D8;
    for (int d = 2 * lane; d < p.D8; d += 2 * kWave) {
      uint32_t x[kPadRows];
#pragma unroll
      for (int i = 0; i < kPadRows; ++i)
        x[i] = d + 1 < p.D ? *reinterpret_cast<const two*>(from[i] + d) : d < p.D ? from[i][d] : 0;
#pragma unroll
      for (int i = 0; i < kPadRows; ++i)
        if (first + i < rows) *reinterpret_cast<uint32_t*>(to + i * p.D8 + d) = x[i];
    }
  }
}

// Results of rows from the shares of their keys: each share's own softmax, weighted by what it holds of the whole.  Lanes hold N elements of a
// row, as few lanes a row as that takes.
template <typename T, int N, int BITS>
__global__ __launch_bounds__(256) void join_forward_kernel(const AttnArgs p, int log_lanes) {
  constexpr int SHARES = 1 << BITS, ITER = N == 4 ? 1 : kLaneCols;
  const int lane = threadIdx.x & 63, lanes = 1 << log_lanes, each = kWave >> log_lanes;
  const int64_t items = static_cast<int64_t>(p.T) * p.H;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * each;
  const int64_t item = min(first + (lane >> log_lanes), items - 1);
  const int row = static_cast<int>(item / p.H), h = static_cast<int>(item - static_cast<int64_t>(row) * p.H);
  const float* from = p.lse_part + static_cast<int64_t>(h) * p.T + row;
  float lse[SHARES], top = kNegInf, sum = 0.0f, acc[ITER][N] = {};
#pragma unroll
  for (int s = 0; s < SHARES; ++s) lse[s] = from[s * items];
#pragma unroll
  for (int s = 0; s < SHARES; ++s) top = fmaxf(top, lse[s]);
#pragma unroll
  for (int s = 0; s < SHARES; ++s) {
    const float w = exp2_f32(lse[s] - top);  // (no share with a finite sum: NaN)
    sum += w;
    const float* part = p.out_part + (s * items + item) * p.D_out;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int d = N * (lane & (lanes - 1)) + 64 * i;
      if (d >= p.D_out) continue;
      if constexpr (N == 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(part + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][j] = fmaf(w, x[j], acc[0][j]);
      } else {
        acc[i][0] = fmaf(w, part[d], acc[i][0]);
      }
    }
  }
  const bool on = top != INFINITY, mine = first + (lane >> log_lanes) < items;  // (infinite: of rows in no sequence, and of no others)
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int d = N * (lane & (lanes - 1)) + 64 * i;
    if (d >= p.D_out || !mine) continue;
#pragma unroll
    for (int j = 0; j < N; ++j) store_result<T>(p, item * p.D_out + d + j, on ? acc[i][j] / sum : 0.0f);
  }
  if (mine && (lane & (lanes - 1)) == 0 && p.lse) p.lse[static_cast<int64_t>(h) * p.T + row] = on ? top + log2f(sum) : INFINITY;
}

// dq, or dk and dv, from their parts, added in order, four elements a lane (n is the number of fours, or of elements where they are no whole fours)
template <typename T, int N>
__global__ __launch_bounds__(256) void join_parts_kernel(const float* __restrict__ dk_part, const float* __restrict__ dv_part,
                                                         T* __restrict__ dk, T* __restrict__ dv, int splits, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const float* part = (blockIdx.y ? dv_part : dk_part) + N * i;
    T* out = (blockIdx.y ? dv : dk) + N * i;
    if constexpr (N == 4) {
      f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
      for (int s = 0; s < splits; ++s) v += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(part + s * n * N));
      if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(out) = v;
      else *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    } else {
      float v = 0.0f;
      for (int s = 0; s < splits; ++s) v += part[s * n];
      store_from_f32<T>(out, v);
    }
  }
}

// the head's padded size and the parts of the other axis that go with it
template <typename Fn>
void with_head(int D, Fn f) {
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, 2> two;
  if (D <= 64) f(std::integral_constant<int, 64>{}, two);
  else if (D <= 96) f(std::integral_constant<int, 96>{}, two);
  else if (D <= 128) f(std::integral_constant<int, 128>{}, two);
  else if (D <= 192) f(std::integral_constant<int, 192>{}, one);  // (twice the rows a tile would take twice the registers for the next one)
  else f(std::integral_constant<int, 256>{}, one);
}

bool in_fours(const AttnArgs& p, bool backward) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  if (backward) bits |= reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.dout);
  // (a tile's rows lie within 32-bit offsets of its first one)
  const int64_t reach = std::max(std::max(p.q_token, p.k_token), std::max<int64_t>(p.v_token, static_cast<int64_t>(p.H) * p.D));
  return bits % 16 == 0 && reach < (1 << 20) && (p.q_token | p.q_head | p.k_token | p.k_head | p.v_token | p.v_head | p.D) % 4 == 0;
}

template <typename K>
void allow_lds(K kernel, size_t bytes, PerDeviceOnce& once) {
  if (bytes <= 65536 || !once.needed()) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  once.done();
}

}  // namespace

void attention_sort_tiles(const AttnArgs& p, int rows, int32_t* query_order, int32_t* key_order, hipStream_t s) {
  hipLaunchKernelGGL(sort_tiles_kernel, dim3(2), dim3(1024), 0, s, p, rows, (p.T + rows - 1) / rows, query_order, key_order);
}

template <int DP, int KW>
void any_forward(const AttnArgs& p, int vec, hipStream_t s) {
  static PerDeviceOnce once;
  allow_lds(any_forward_kernel<DP, KW>, kAnyLds<DP, KW>, once);
  const int rows = 64 / KW, tiles = (p.T + rows - 1) / rows;
  hipLaunchKernelGGL((any_forward_kernel<DP, KW>), dim3((tiles * p.H) << p.share_bits), dim3(256), (kAnyLds<DP, KW>), s, p, tiles, vec);
}

int attention_any_rows(int D) { return D <= 128 ? 32 : 64; }

void attention_any_forward(const AttnArgs& p, hipStream_t s) {
  const int vec = in_fours(p, false);
  with_head(p.D, [&](auto d, auto parts) { any_forward<decltype(d)::value, decltype(parts)::value>(p, vec, s); });
}

template <int DP, int KW>
void any_backward(const AttnArgs& p, int vec, hipStream_t s) {
  static PerDeviceOnce once_q, once_kv;
  allow_lds(any_dq_kernel<DP, KW>, kAnyLds<DP, KW>, once_q);
  allow_lds(any_dkv_kernel<DP, KW>, kAnyLds<DP, KW>, once_kv);
  const int rows = 64 / KW, tiles = (p.T + rows - 1) / rows;
  hipLaunchKernelGGL((any_dq_kernel<DP, KW>), dim3((tiles * p.H) << p.share_bits), dim3(256), (kAnyLds<DP, KW>), s, p, tiles, vec);
  hipLaunchKernelGGL((any_dkv_kernel<DP, KW>), dim3(tiles * p.G * p.splits), dim3(256), (kAnyLds<DP, KW>), s, p, tiles, vec);
}

template <typename T>
void join_parts(const AttnArgs& p, hipStream_t s) {
  auto join = [&](const float* a_part, const float* b_part, void* a, void* b, int heads, int parts) {
    if (parts <= 1) return;
    const int64_t n = static_cast<int64_t>(p.T) * heads * p.D_out;
    const bool fours = n % 4 == 0 && (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % (4 * sizeof(T)) == 0;
    const int64_t items = fours ? n / 4 : n;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((items + 255) / 256, 1 << 20)), b ? 2 : 1);
    if (fours) hipLaunchKernelGGL((join_parts_kernel<T, 4>), grid, dim3(256), 0, s, a_part, b_part, static_cast<T*>(a), static_cast<T*>(b), parts, items);
    else hipLaunchKernelGGL((join_parts_kernel<T, 1>), grid, dim3(256), 0, s, a_part, b_part, static_cast<T*>(a), static_cast<T*>(b), parts, items);
  };
  join(p.dq_part, nullptr, p.dq, nullptr, p.H, 1 << p.share_bits);
  join(p.dk_part, p.dv_part, p.dk, p.dv, p.G, p.splits);
}

template <typename T, int N>
void join_forward(const AttnArgs& p, hipStream_t s) {
  int log_lanes = 0;
  while (N << log_lanes < p.D_out && log_lanes < 6) ++log_lanes;
  const int64_t each = 4 * (kWave >> log_lanes), items = static_cast<int64_t>(p.T) * p.H;
  const dim3 grid(static_cast<unsigned>((items + each - 1) / each));  // (at most 1024 x 128 rows, or there are no shares)
  if (p.share_bits == 1) hipLaunchKernelGGL((join_forward_kernel<T, N, 1>), grid, dim3(256), 0, s, p, log_lanes);
  else if (p.share_bits == 2) hipLaunchKernelGGL((join_forward_kernel<T, N, 2>), grid, dim3(256), 0, s, p, log_lanes);
  else hipLaunchKernelGGL((join_forward_kernel<T, N, 3>), grid, dim3(256), 0, s, p, log_lanes);
}
template <typename T>
void join_forward(const AttnArgs& p, hipStream_t s) {
  if (p.D_out % 4 == 0) join_forward<T, 4>(p, s);
  else join_forward<T, 1>(p, s);
}

void attention_any_backward(const AttnArgs& p, hipStream_t s) {
  const int vec = in_fours(p, true);
  with_head(p.D, [&](auto d, auto parts) { any_backward<decltype(d)::value, decltype(parts)::value>(p, vec, s); });
}

}  // namespace mi355

using namespace mi355;

namespace {

int check_attention(const char* what, int dtype, int64_t sequences, int64_t T, int64_t H, int64_t G, int64_t D, float scale) {
  MI355_REQUIRE(dtype == MI355_F32 || dtype == MI355_BF16, "%s: dtype %d is neither fp32 nor bf16", what, dtype);
  MI355_REQUIRE(T >= 0 && T < (1ll << 30) && sequences >= 0 && sequences < (1ll << 30), "%s: bad shape tokens=%lld sequences=%lld", what,
                (long long)T, (long long)sequences);
  MI355_REQUIRE(H >= 1 && G >= 1 && H <= 65535 && H % G == 0, "%s: %lld query heads are no multiple of %lld key heads", what,
                (long long)H, (long long)G);
  // (2^24 workgroups of 256 lanes a launch)
  MI355_REQUIRE((T + 127) / 128 * H < (1ll << (dtype == MI355_BF16 ? 24 : 22)), "%s: %lld tokens of %lld heads are too many for one launch", what,
                (long long)T, (long long)H);
  MI355_REQUIRE(H * ((D + 7) / 8 * 8) < (1 << 22), "%s: %lld heads of %lld are too many", what, (long long)H, (long long)D);
  MI355_REQUIRE(D >= 1 && D <= kHeadMax, "%s: head size %lld is not within 1 to %d", what, (long long)D, kHeadMax);
  // (lse over scale log2(e), which the backward starts its sums from, stays a number)
  MI355_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f, "%s: the scale must be finite and positive, from 2^-100 to 2^100", what);
  return MI355_OK;
}

// Parts of a key head's group of query heads: as many as it takes to give every CU two workgroups, and up to four for shares that can be
// evened out.  Parts cost a trip of dk and dv through memory in fp32.  Tiles of 128 keys, 32/4 heads of 128, us, dk/dv and joining the
// parts: 8192 rows in 4 sequences 2 parts 398 + 20, 4 294 + 37, 8 322 + 89; 16384 in 11 1 1221, 2 692 + 49, 4 598 + 85.
int head_parts(int64_t T, int64_t H, int64_t G) {
  const int64_t group = H / G, tiles = (T + 127) / 128 * G;
  const int64_t parts = std::min(group, std::max((kHeldAtOnce + tiles - 1) / tiles, std::min<int64_t>(4, (2048 + tiles - 1) / tiles)));
  const int64_t heads = (group + parts - 1) / parts;
  return (int)((group + heads - 1) / heads);
}

// Where tiles are too few to fill the card, each one's other axis is dealt over workgroups (1 << bits of them, up to eight), whose parts are joined
// through memory in fp32.  Whether that pays is a matter of what a workgroup of its own takes against the trip: of `products` per key, a
// workgroup alone reaches two thirds of the matrix rate of its CU, and the card no more than the whole of it; a launch that joins 3 us; memory 5 TB/s.
// One sequence, bf16 heads of 128, us, whole / dealt: forward of 16384 rows of one head 287 / 101, 4096 of 4 77 / 42, 1024 of 4 24 / 19 (of 16 25 / 30: not
// dealt); backward 1060 / 305, 292 / 126, 90 / 54 (of 16 99 / 74); fp32, 4096 of one 223 / 80 and 664 / 216.  (Drawn with earlier kernels; dealt, these are
// 97, 40, 19, 298, 124, 54 and 77, 82 and 219 now.)
int tile_rows(int64_t D, int dtype) { return dtype == MI355_BF16 ? attention_bf16_rows() : attention_any_rows((int)D); }
int64_t tiles_of(int64_t T, int64_t D, int dtype) { return (T + tile_rows(D, dtype) - 1) / tile_rows(D, dtype); }
constexpr int kMostShares = 3;  // a power of two
// as many as there can be, of sequences of any length
int most_share_bits(int64_t workgroups, int64_t T) {
  int bits = 0;
  while (bits < kMostShares && workgroups << (bits + 1) <= 2 * kHeldAtOnce && T >= 64 << (bits + 1)) ++bits;
  return bits;
}
// `part`: elements that a share writes and its joining reads; `parts`: those of other cuts, joined in any case if there are several
int share_bits(int64_t workgroups, int products, int64_t T, int64_t sequences, int64_t D, int dtype, int64_t part, int64_t parts) {
  const double rate = dtype == MI355_BF16 ? 1200e6 / 256 : 137e6 / 256;  // flops a us and CU
  const double keys = static_cast<double>(T) / std::max<int64_t>(sequences, 1), whole = keys * products * 2.0 * tile_rows(D, dtype) * D / rate;
  auto time = [&](int bits) {
    const double rounds = static_cast<double>(workgroups) / kHeldAtOnce;  // (a tile's rows see half of the keys on average, and two are held by a CU)
    return whole * std::max(1.5 / (1 << bits), rounds) + (bits && parts == 1 ? 3.0 : 0.0) + ((parts << bits) > 1 ? 8e-6 / 5 * part * (parts << bits) : 0.0);
  };
  int best = 0;
  for (int bits = 1; bits <= most_share_bits(workgroups, T); ++bits) {
    // fp32 workgroups hold a CU's registers, those of heads beyond 96 all of them: more than 512 end later (4096 rows of a head of 128 in 1024 109 us, in
    // 512 85; of 4 heads 268 and 242), but smaller heads' 512 end sooner as halves (4 of 64: backward 518 -> 366)
    if (dtype == MI355_F32 && (bits > 1 || D > 96) && workgroups << bits > kHeldAtOnce) break;
    if (time(bits) < 0.95 * time(best)) best = bits;
  }
  return best;
}
int forward_bits(int64_t T, int64_t H, int64_t D, int64_t sequences, int dtype) {
  return share_bits(tiles_of(T, D, dtype) * H, 2, T, sequences, D, dtype, T * H * D, 1);
}
// What a call's launches are, by its sizes alone
struct AttnPaths {
  bool sorted, bwd_sorted;  // tiles in the order of their work: in the forward, in the backward
  int bits, dq_bits;      // shares of the keys: 1 << bits in the forward, 1 << dq_bits for dq
  int parts, key_bits;    // of dk and dv: parts of the group of query heads, times 1 << key_bits shares of the queries
};
AttnPaths paths_of(int64_t T, int64_t H, int64_t G, int64_t D, int64_t sequences, int dtype) {
  const int64_t tiles = tiles_of(T, D, dtype);
  AttnPaths x;
  x.sorted = sorted_tiles(sequences, T, tiles, H, kLongForward), x.bwd_sorted = sorted_tiles(sequences, T, tiles, H, kLongBackward);
  x.bits = forward_bits(T, H, D, sequences, dtype);
  x.dq_bits = share_bits(tiles * H, 3, T, sequences, D, dtype, T * H * D, 1);
  x.parts = head_parts(T, H, G);
  x.key_bits = share_bits(tiles * G * x.parts, 4, T, sequences, D, dtype, 2 * T * G * D, x.parts);
  return x;
}
int64_t out_part_bytes(int64_t T, int64_t H, int64_t D, int bits) {
  return bits ? ((4 * T * H * D << bits) + 15) / 16 * 16 : 0;
}
int64_t lse_part_bytes(int64_t T, int64_t H, int bits) { return bits ? ((4 * T * H << bits) + 15) / 16 * 16 : 0; }

AttnArgs attention_args(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head, const void* v,
                        int64_t v_token, int64_t v_head, const int32_t* cu, int64_t sequences, float scale, int64_t T, int64_t H,
                        int64_t G, int64_t D) {
  AttnArgs p = {};
  p.q = q, p.k = k, p.v = v;
  p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
  p.cu = cu, p.sequences = (int)sequences;
  p.T = (int)T, p.H = (int)H, p.G = (int)G, p.D = (int)D, p.group = (int)(H / G);
  p.scale = scale, p.c = (float)(scale * 1.4426950408889634);
  p.D_out = (int)D;
  return p;
}

// an order of the tiles, in whole pieces of 16 bytes
int64_t order_bytes(int64_t T) { return ((T + kLeastRows - 1) / kLeastRows + 3) / 4 * 16; }

bool padded_heads(int64_t D, int dtype) { return dtype == MI355_BF16 && D % 8 != 0; }
int64_t padded_bytes(int64_t T, int64_t heads, int64_t D) { return T * heads * ((D + 7) / 8 * 8) * 2; }

// Lets p's q, k and v (and dout, out and its rest) be padded copies in `space`.
void pad_heads(AttnArgs& p, bool backward, void* space, hipStream_t s) {
  AttnArgs q = p;
  PadArgs a = {};
  a.T = p.T, a.D = p.D, a.D8 = (p.D + 7) / 8 * 8;
  uint16_t* at = static_cast<uint16_t*>(space);
  int n = 0;
  auto add = [&](const void*& x, int64_t token, int64_t head, int heads) {
    a.from[n] = static_cast<const uint16_t*>(x), a.to[n] = at, a.token[n] = token, a.head[n] = head, a.heads[n] = heads;
    x = at;
    at += static_cast<int64_t>(p.T) * heads * a.D8;
    ++n;
  };
  const int64_t dense = static_cast<int64_t>(p.H) * p.D;
  add(q.q, p.q_token, p.q_head, p.H);
  add(q.k, p.k_token, p.k_head, p.G);
  add(q.v, p.v_token, p.v_head, p.G);
  if (backward) {
    add(q.dout, dense, p.D, p.H);
    add(q.o, dense, p.D, p.H);
    const void* rest = p.rest;
    if (rest) add(rest, dense, p.D, p.H);
    q.rest = const_cast<void*>(rest);
  }
  q.D = a.D8;
  q.q_token = static_cast<int64_t>(p.H) * a.D8, q.k_token = q.v_token = static_cast<int64_t>(p.G) * a.D8;
  q.q_head = q.k_head = q.v_head = a.D8;
  const int64_t blocks = std::min<int64_t>((static_cast<int64_t>(p.T) * p.H + 4 * kPadRows - 1) / (4 * kPadRows), 1 << 22);
  hipLaunchKernelGGL(pad_heads_kernel, dim3((unsigned)blocks, n), dim3(256), 0, s, a);
  p = q;
}

}  // namespace

extern "C" int mi355_varlen_attention_fwd(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                          int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                          int64_t v_head_stride, int dtype, const int32_t* cu_seqlens, int64_t sequences, float scale,
                                          void* out, void* out_rest, float* lse, void* workspace, int64_t T, int64_t H,
                                          int64_t G, int64_t D, void* stream) {
  if (int rc = check_attention("varlen_attention_fwd", dtype, sequences, T, H, G, D, scale)) return rc;
  if (T == 0) return MI355_OK;
  MI355_REQUIRE(q && k && v && cu_seqlens && out, "varlen_attention_fwd: null pointer");
  AttnArgs p = attention_args(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride,
                              cu_seqlens, sequences, scale, T, H, G, D);
  p.out = out, p.lse = lse, p.rest = dtype == MI355_BF16 ? out_rest : nullptr;
  MI355_REQUIRE(aligned16(workspace), "varlen_attention_fwd: the workspace must start on a 16-byte boundary");
  const bool matrix = dtype == MI355_BF16, padded = padded_heads(D, dtype);
  MI355_REQUIRE(!padded || workspace, "varlen_attention_fwd: workspace required for bf16 heads of %lld elements", (long long)D);
  if (padded) pad_heads(p, false, static_cast<char*>(workspace) + order_bytes(T), as_stream(stream));
  MI355_REQUIRE(!matrix || attention_bf16_covers(p), "varlen_attention_fwd: bf16 operands must start and stride in whole pieces of 16 bytes");
  const AttnPaths paths = paths_of(T, H, G, D, sequences, dtype);
  if (workspace && paths.sorted) {
    attention_sort_tiles(p, matrix ? attention_bf16_rows() : attention_any_rows((int)D), static_cast<int32_t*>(workspace), nullptr, as_stream(stream));
    p.query_order = static_cast<int32_t*>(workspace);
  }
  if (workspace) p.share_bits = paths.bits;
  if (p.share_bits) {
    char* at = static_cast<char*>(workspace) + order_bytes(T) + (padded ? padded_bytes(T, H + 2 * G, D) : 0);
    p.out_part = reinterpret_cast<float*>(at);
    p.lse_part = reinterpret_cast<float*>(at + out_part_bytes(T, H, D, p.share_bits));
  }
  if (matrix) attention_bf16_forward(p, as_stream(stream));
  else attention_any_forward(p, as_stream(stream));
  if (p.share_bits) matrix ? join_forward<uint16_t>(p, as_stream(stream)) : join_forward<float>(p, as_stream(stream));
  return check_launch("varlen_attention_fwd");
}

extern "C" int mi355_varlen_attention_paths(int64_t T, int64_t H, int64_t G, int64_t D, int64_t sequences, int dtype) {
  if (T < 1 || check_attention("varlen_attention_paths", dtype, sequences, T, H, G, D, 1.0f)) return 0;
  const AttnPaths x = paths_of(T, H, G, D, sequences, dtype);
  return (x.sorted ? MI355_ATTENTION_FWD_SORTED : 0) | (x.bwd_sorted ? MI355_ATTENTION_BWD_SORTED : 0) | x.bits << 4 | x.dq_bits << 8 | x.key_bits << 12 | x.parts << 16;
}

extern "C" int64_t mi355_varlen_attention_fwd_workspace_bytes(int64_t T, int64_t H, int64_t G, int64_t D, int64_t sequences, int dtype) {
  if (T < 1 || H < 1 || G < 1 || D < 1) return 0;
  const int bits = forward_bits(T, H, D, sequences, dtype);
  const int64_t copies = padded_heads(D, dtype) ? padded_bytes(T, H + 2 * G, D) : 0;
  if (!copies && !bits && !sorted_tiles(sequences, T, tiles_of(T, D, dtype), H, kLongForward)) return 0;
  return order_bytes(T) + copies + out_part_bytes(T, H, D, bits) + lse_part_bytes(T, H, bits);
}

extern "C" int64_t mi355_varlen_attention_bwd_workspace_bytes(int64_t T, int64_t H, int64_t G, int64_t D, int dtype) {
  if (T < 1 || H < 1 || G < 1 || H % G || D < 1) return 0;
  const int64_t parts = head_parts(T, H, G), tiles = tiles_of(T, D, dtype);
  const int bits = most_share_bits(tiles * H, T);
  const int64_t key_parts = parts << most_share_bits(tiles * G * parts, T);
  return 4 * ((2 * H * T + 3) / 4 * 4) + 2 * order_bytes(T) + (padded_heads(D, dtype) ? padded_bytes(T, 4 * H + 2 * G, D) : 0) +
         out_part_bytes(T, H, D, bits) + (key_parts > 1 ? 8 * key_parts * T * G * D : 0);
}

extern "C" int mi355_varlen_attention_bwd(const void* dout, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                          int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                          int64_t v_head_stride, const void* out, const void* out_rest, const float* lse,
                                          int dtype, const int32_t* cu_seqlens, int64_t sequences, float scale, void* dq, void* dk, void* dv,
                                          void* workspace, int64_t T, int64_t H, int64_t G, int64_t D, void* stream) {
  if (int rc = check_attention("varlen_attention_bwd", dtype, sequences, T, H, G, D, scale)) return rc;
  if (T == 0) return MI355_OK;
  MI355_REQUIRE(dout && q && k && v && out && lse && cu_seqlens && dq && dk && dv && workspace, "varlen_attention_bwd: null pointer");
  MI355_REQUIRE(aligned16(workspace), "varlen_attention_bwd: the workspace must start on a 16-byte boundary");
  AttnArgs p = attention_args(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride,
                              cu_seqlens, sequences, scale, T, H, G, D);
  p.o = out, p.rest = dtype == MI355_BF16 ? const_cast<void*>(out_rest) : nullptr;
  p.dout = dout, p.lse = const_cast<float*>(lse), p.dq = dq, p.dk = dk, p.dv = dv;
  const AttnPaths paths = paths_of(T, H, G, D, sequences, dtype);
  p.share_bits = paths.dq_bits, p.key_share_bits = paths.key_bits, p.splits = paths.parts << paths.key_bits;
  p.delta = static_cast<float*>(workspace);
  char* at = reinterpret_cast<char*>(p.delta + (2 * H * T + 3) / 4 * 4);
  int32_t *query_order = reinterpret_cast<int32_t*>(at), *key_order = reinterpret_cast<int32_t*>(at + order_bytes(T));
  at += 2 * order_bytes(T);
  if (padded_heads(D, dtype)) {
    pad_heads(p, true, at, as_stream(stream));
    at += padded_bytes(T, 4 * H + 2 * G, D);
  }
  p.dq_part = reinterpret_cast<float*>(at);
  at += out_part_bytes(T, H, D, p.share_bits);
  p.dk_part = reinterpret_cast<float*>(at);
  p.dv_part = p.dk_part + static_cast<int64_t>(p.splits) * T * G * D;
  const bool matrix = dtype == MI355_BF16;
  MI355_REQUIRE(!matrix || attention_bf16_covers(p), "varlen_attention_bwd: bf16 operands must start and stride in whole pieces of 16 bytes");
  if (paths.bwd_sorted) {
    attention_sort_tiles(p, matrix ? attention_bf16_rows() : attention_any_rows((int)D), query_order, key_order, as_stream(stream));
    p.query_order = query_order, p.key_order = key_order;
  }
  if (matrix) attention_bf16_backward(p, as_stream(stream));
  else attention_any_backward(p, as_stream(stream));
  if (dtype == MI355_F32) join_parts<float>(p, as_stream(stream));
  else join_parts<uint16_t>(p, as_stream(stream));
  return check_launch("varlen_attention_bwd");
}
