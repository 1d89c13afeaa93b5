// What the attention kernels share: their arguments, the sequence of a row, and the careful row-by-row forms for what a
// value that is not finite has spoilt.
//
// Causal attention over sequences packed one behind another, for query head h on key head h / (H / G):
//   s_rj = q_r . k_j,   p_rj = exp2(c s_rj - lse_r) for start(r) <= j <= r,   o_r = sum_j p_rj v_j
// with c = scale log2(e) and lse_r = log2 sum_j exp2(c s_rj); and backward, with delta_r = do_r . o_r,
//   ds_rj = p_rj (do_r . v_j - delta_r) scale,
//   dq_r = sum_j ds_rj k_j,   dk_j = sum_h,r ds_rj q_r,   dv_j = sum_h,r p_rj do_r.
//
// Tiles are runs of rows of the packed tensors, whatever sequences they cut through: a tile of many short sequences is
// then as full as one of a long one, and the grid follows from the sizes alone, without reading cu_seqlens back.  Every row looks
// up its own sequence; the look-up's answer holds start <= row < end whatever the array holds, so no index leaves the tensors.
//
// Rows whose mask leaves nothing (in no sequence) get zeros.  A matrix product cannot leave out an element:
// 0 x NaN, of a value in a masked place of the same tile, is NaN in the sum.  Such a sum shows at the end
// as NaN, and only then the row is formed again by the functions here, key by key, without the masked ones.  Where no input is
// NaN or infinite that costs one comparison an element of the result.
#pragma once
#include "bf16_tiles.h"
#include "common.h"

namespace mi355 {

struct AttnArgs {
  const void *q, *k, *v;  // (T, H, D), (T, G, D), (T, G, D); elements of a head contiguous
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, in elements
  void* out;              // (T, H, D) dense
  float* lse;             // (H, T), log2
  void* rest;             // (T, H, D) dense, bf16 only: what rounding took from out (written forward, read backward); null: not kept
  // backward
  const void *o, *dout;   // (T, H, D) dense
  float* delta;           // (H, T), negated by the bf16 kernels, which put -lse / c behind it (2 H, T)
  void *dq, *dk, *dv;     // dense; (splits > 1: dk_part, dv_part instead of dk, dv)
  float *dk_part, *dv_part;  // [splits][T][G][D] fp32
  // tiles whose other axis is dealt over 1 << share_bits workgroups (queries) or 1 << key_share_bits (keys): parts in fp32, joined behind them
  int share_bits, key_share_bits;
  float *out_part, *lse_part, *dq_part;  // [shares][T][H][D], [shares][H][T], [shares][T][H][D]
  const int32_t* cu;      // [sequences + 1]
  int sequences;
  int T, H, G, D, group;  // group = H / G
  int D_out;              // elements of a head in results and their parts: D, or fewer where the operands are copies padded to D
  int splits;             // parts of dk and dv: those a key head's group of query heads is cut into, times 1 << key_share_bits
  float scale, c;         // c = scale log2(e)
  // tiles of rows by descending work, for the kernels whose rows are queries and for dk and dv; null: as they lie, the last (first) tile first
  const int32_t *query_order, *key_order;
};

constexpr float kNegInf = -INFINITY;

// A kernel's arguments (AttnArgs its first) as memory to be read from here on.  What a kernel needs behind its loop only, and the careful
// forms at its end above all, is otherwise fetched and prepared in front of it, and held in registers that the loop has no room for.
__device__ __forceinline__ const AttnArgs& late_arguments() {
  uint64_t at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(at));
  return *(const AttnArgs*)reinterpret_cast<const __attribute__((address_space(4))) AttnArgs*>(at);
}

// The sequence [start, end) that a row lies in, or start = end = 0.  The entries on both sides of the answer have been compared with the
// row, so start <= row < end however the array is ordered; clamped to the rows there are.
__device__ __forceinline__ void sequence_of(const int32_t* cu, int sequences, int T, int row, int& start, int& end) {
  int a = 0, b = sequences + 1;  // entries below a are <= row, entries from b on are > row
  while (a < b) {
    const int mid = (a + b) >> 1;
    if (cu[mid] <= row) a = mid + 1;
    else b = mid;
  }
  start = end = 0;
  if (a == 0 || a > sequences || row >= T) return;
  start = max(cu[a - 1], 0);
  end = min(cu[a], T);
}

// Narrows [lo, hi) to the steps that fall to one of 1 << bits workgroups.
__device__ __forceinline__ void take_share(int& lo, int& hi, int step, int share, int bits) {
  const int from = lo, steps = lo < hi ? (hi - lo + step - 1) / step : 0;
  lo = from + ((steps * share) >> bits) * step;
  hi = min(hi, from + ((steps * (share + 1)) >> bits) * step);
}

// Order of a stretch of code, N times: a matrix instruction, READS reads of LDS, VALU vector instructions
template <int N, int READS, int VALU>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (READS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if (VALU) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
  }
}
template <int READS>
__device__ __forceinline__ void reads_first() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
}

struct Place {
  int head, tile;
};
// Workgroup b runs on XCD b % 8.  Heads that share keys go to one XCD, whose L2 then holds them once; tiles in their sorted order, or
// as they lie, `last` first.
__device__ __forceinline__ Place place_of(int block, int heads, int tiles, const int32_t* order, bool last) {
  Place w;
  int rank;
  if (heads % 8 == 0) {
    const int each = heads / 8, j = block >> 3;
    w.head = (block & 7) * each + j % each;
    rank = j / each;
  } else {
    w.head = block % heads;
    rank = block / heads;
  }
  w.tile = order ? order[rank] : last ? tiles - 1 - rank : rank;
  return w;
}

__device__ __forceinline__ float exp2_f32(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T>
__device__ __forceinline__ const T* row_at(const void* base, int64_t token, int64_t head, int64_t t, int64_t h) {
  return static_cast<const T*>(base) + t * token + h * head;
}

// an element of the forward's result, and what its rounding took
template <typename T>
__device__ __forceinline__ void store_result(const AttnArgs& p, int64_t at, float v) {
  T* out = static_cast<T*>(p.out) + at;
  store_from_f32<T>(out, v);
  if constexpr (sizeof(T) == 2)
    if (p.rest) static_cast<uint16_t*>(p.rest)[at] = f32_to_bf16(v - round_bf16(v));
}

// ---- one row by one wave: lanes over keys (or queries) for the products, over the head's elements for the sums -------------------
constexpr int kHeadMax = 256;          // elements of a head
constexpr int kLaneCols = kHeadMax / 64;

// sum_d a[d] b[d], a wave's lanes each with rows of their own
template <typename T>
__device__ float careful_dot(const T* a, const T* b, int D) {
  float s = 0.0f;
  for (int d = 0; d < D; ++d) s = fmaf(load_as_f32<T>(a + d), load_as_f32<T>(b + d), s);
  return s;
}

template <typename T>
__device__ __forceinline__ void careful_forward_row(const AttnArgs& p, int h, int row, int start) {
  const int lane = threadIdx.x & 63;
  const T* q = row_at<T>(p.q, p.q_token, p.q_head, row, h);
  float acc[kLaneCols] = {}, m = kNegInf, l = 0.0f;
  for (int j0 = start; j0 <= row; j0 += kWave) {
    const int j = j0 + lane;
    const float s = j <= row ? careful_dot<T>(q, row_at<T>(p.k, p.k_token, p.k_head, j, h / p.group), p.D) : kNegInf;
    const float top = fmaxf(m, wave_max(s)), ref = top == kNegInf ? 0.0f : top * p.c;
    const float w = j <= row ? exp2_f32(fmaf(s, p.c, -ref)) : 0.0f, keep = m == kNegInf ? 0.0f : exp2_f32(m * p.c - ref);
    l = l * keep + wave_sum(w);
#pragma unroll
    for (int i = 0; i < kLaneCols; ++i) acc[i] *= keep;
    for (int n = 0; n < kWave && j0 + n <= row; ++n) {
      const float wn = __shfl(w, n, kWave);
      const T* v = row_at<T>(p.v, p.v_token, p.v_head, j0 + n, h / p.group);
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i)
        if (lane + 64 * i < p.D) acc[i] = fmaf(wn, load_as_f32<T>(v + lane + 64 * i), acc[i]);
    }
    m = top;
  }
  const int64_t dense = (static_cast<int64_t>(row) * p.H + h) * p.D_out;
#pragma unroll
  for (int i = 0; i < kLaneCols; ++i)
    if (lane + 64 * i < p.D_out) store_result<T>(p, dense + lane + 64 * i, acc[i] / l);
}

// dq of one row over the keys of [from, to), into the part `share` where there are parts
template <typename T>
__device__ __forceinline__ void careful_dq_row(const AttnArgs& p, int h, int row, int start, float lse, float delta, int from, int to, int share) {
  const int lane = threadIdx.x & 63;
  const T* q = row_at<T>(p.q, p.q_token, p.q_head, row, h);
  const T* dout = static_cast<const T*>(p.dout) + (static_cast<int64_t>(row) * p.H + h) * p.D;
  float acc[kLaneCols] = {};
  to = min(to, row + 1);
  for (int j0 = max(start, from); j0 < to; j0 += kWave) {
    const int j = j0 + lane;
    float ds = 0.0f;
    if (j < to && start < row) {
      const float w = exp2_f32(fmaf(careful_dot<T>(q, row_at<T>(p.k, p.k_token, p.k_head, j, h / p.group), p.D), p.c, -lse));
      ds = w * (careful_dot<T>(dout, row_at<T>(p.v, p.v_token, p.v_head, j, h / p.group), p.D) - delta);
    }
    for (int n = 0; n < kWave && j0 + n < to; ++n) {
      const float dn = __shfl(ds, n, kWave);
      const T* k = row_at<T>(p.k, p.k_token, p.k_head, j0 + n, h / p.group);
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i)
        if (lane + 64 * i < p.D) acc[i] = fmaf(dn, load_as_f32<T>(k + lane + 64 * i), acc[i]);
    }
  }
  const int64_t at = (static_cast<int64_t>(row) * p.H + h) * p.D_out, part = static_cast<int64_t>(share) * p.T * p.H * p.D_out + at;
#pragma unroll
  for (int i = 0; i < kLaneCols; ++i) {
    const int d = lane + 64 * i;
    if (d >= p.D_out) continue;
    if (p.share_bits) p.dq_part[part + d] = acc[i] * p.scale;
    else store_from_f32<T>(static_cast<T*>(p.dq) + at + d, acc[i] * p.scale);
  }
}

// dk and dv of one key over the rows of [from, to) of the query heads [h0, h1), into the part `split` where there are parts; delta is kept
// times `sign`
template <typename T>
__device__ __forceinline__ void careful_dkv_row(const AttnArgs& p, int g, int key, int start, int end, int h0, int h1, int from, int to, int split,
                                                float sign) {
  const int lane = threadIdx.x & 63;
  const T* k = row_at<T>(p.k, p.k_token, p.k_head, key, g);
  const T* v = row_at<T>(p.v, p.v_token, p.v_head, key, g);
  float dk[kLaneCols] = {}, dv[kLaneCols] = {};
  end = min(end, to);
  for (int h = h0; h < h1; ++h) {
    for (int r0 = max(key, from); r0 < end; r0 += kWave) {
      const int r = r0 + lane;
      float w = 0.0f, ds = 0.0f;
      if (r < end) {
        const T* dout = static_cast<const T*>(p.dout) + (static_cast<int64_t>(r) * p.H + h) * p.D;
        const int64_t at = static_cast<int64_t>(h) * p.T + r;
        w = exp2_f32(fmaf(careful_dot<T>(row_at<T>(p.q, p.q_token, p.q_head, r, h), k, p.D), p.c, -p.lse[at]));
        ds = start < r ? w * (careful_dot<T>(dout, v, p.D) - sign * p.delta[at]) : 0.0f;
      }
      for (int n = 0; n < kWave && r0 + n < end; ++n) {
        const float wn = __shfl(w, n, kWave), dn = __shfl(ds, n, kWave);
        const T* q = row_at<T>(p.q, p.q_token, p.q_head, r0 + n, h);
        const T* dout = static_cast<const T*>(p.dout) + (static_cast<int64_t>(r0 + n) * p.H + h) * p.D;
#pragma unroll
        for (int i = 0; i < kLaneCols; ++i)
          if (lane + 64 * i < p.D) {
            dv[i] = fmaf(wn, load_as_f32<T>(dout + lane + 64 * i), dv[i]);
            dk[i] = fmaf(dn, load_as_f32<T>(q + lane + 64 * i), dk[i]);
          }
      }
    }
  }
  const int64_t at = (static_cast<int64_t>(key) * p.G + g) * p.D_out, part = static_cast<int64_t>(split) * p.T * p.G * p.D_out + at;
#pragma unroll
  for (int i = 0; i < kLaneCols; ++i) {
    const int d = lane + 64 * i;
    if (d >= p.D_out) continue;
    if (p.splits > 1) {
      p.dk_part[part + d] = dk[i] * p.scale;
      p.dv_part[part + d] = dv[i];
    } else {
      store_from_f32<T>(static_cast<T*>(p.dk) + at + d, dk[i] * p.scale);
      store_from_f32<T>(static_cast<T*>(p.dv) + at + d, dv[i]);
    }
  }
}

// ---- order of the tiles ---------------------------------------------------------------------------------
// A tile's work is as long as the other axis that its rows see.  Of one sequence the last rows see the most; of several nothing about
// it is known without cu_seqlens, and a heavy tile that starts last ends long after the others.  Where there are more
// workgroups than the card holds at once and sequences are long on average, one small kernel (5 us) sorts the tiles by their work
// first: forward and dq of 8192 rows in 4 sequences, 32 heads of 128, 178 -> 164 and 260 -> 239 us, of 16384 in 11 345 -> 318 and 502 -> 462.
constexpr int kHeldAtOnce = 512;     // workgroups: two a CU
constexpr int kLongOnAverage = 512;  // rows a sequence: below, a tile's work differs by less than the sorting costs
inline bool sorted_tiles(int64_t sequences, int64_t T, int64_t tiles, int64_t heads) {
  return sequences > 1 && T >= kLongOnAverage * sequences && tiles * heads > kHeldAtOnce / 2;
}
// order[i]: the i-th tile of `rows` rows to start
void attention_sort_tiles(const AttnArgs& p, int rows, int32_t* query_order, int32_t* key_order, hipStream_t s);

// ---- launches, by file --------------------------------------------------------------------------------
constexpr int kLeastRows = 32;  // rows of a tile, at least
int attention_any_rows(int D);
int attention_bf16_rows();
void attention_any_forward(const AttnArgs& p, hipStream_t s);
void attention_any_backward(const AttnArgs& p, hipStream_t s);
bool attention_bf16_covers(const AttnArgs& p);
void attention_bf16_forward(const AttnArgs& p, hipStream_t s);
void attention_bf16_backward(const AttnArgs& p, hipStream_t s);

}  // namespace mi355
