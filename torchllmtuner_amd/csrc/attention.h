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
// 0 x NaN, of a value in a masked place of the same tile, is NaN in the sum.  Rows of the other axis outside [lo, hi), which no row of the
// workgroup sees, are therefore never fetched; what is left are the tiles in which a wave's rows see different things: around the diagonal
// and where sequences meet.  Such a sum shows at the end as NaN, and the row is formed again by the functions here, key by key,
// without the masked ones.  So does the sum of a row that sees the NaN itself, of which there may be as many as rows: not formed
// again are rows whose statistics are NaN, and rows whose masked places, searched once a wave, hold nothing that is not finite; the others
// begin with the nearest keys and end as soon as every spoilt element is NaN by itself.  Where no input is NaN or
// infinite that costs one comparison an element of the result.  A training step of 4096 rows in two sequences and 96 behind, 8/2 heads of 128,
// bf16 (fp32): 0.25 ms (1.2); all NaN 0.9 (2.0), rows behind NaN 0.25 (1.2), one query NaN 1.0 (2.0), the second sequence NaN, next to
// whose first rows the last 56 of the first one lie in tiles with masked places only: 2.9 (3.9), which grows with the length of theirs.
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

// ---- rows formed again ---------------------------------------------------------------------------------
constexpr int kHeadMax = 256;          // elements of a head
constexpr int kLaneCols = kHeadMax / 64;

struct Span {
  int lo, hi;
};
// Of the tiles of `step` rows from lo on up to hi: those within [from, to), which have no masked place.  Empty, at lo, where there are none.
__device__ __forceinline__ Span whole_tiles(int lo, int hi, int step, int from, int to) {
  const Span s = {lo + (max(from - lo, 0) + step - 1) / step * step, lo + max(min(to, hi) - lo, 0) / step * step};
  return s.lo < s.hi ? s : Span{lo, lo};
}

// the lane, formed anew where a kernel has no register to keep it in
__device__ __forceinline__ int lane_anew() { return opaque(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0))); }

// Widens `at` to the first and last of a head's rows [from, to) that hold something NaN or infinite
template <typename T>
__device__ __forceinline__ void find_not_finite(const T* base, int64_t token, int from, int to, int D, Span& at) {
  const int lane = lane_anew();
  for (int r0 = from; r0 < to; r0 += 8) {  // (eight rows' loads under way together)
    bool bad[8] = {};
    for (int d = lane; d < D; d += kWave)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = load_as_f32<T>(base + min(r0 + i, to - 1) * token + d);
        bad[i] |= x - x != 0.0f;
      }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (__any(bad[i])) at.lo = min(at.lo, r0 + i), at.hi = max(at.hi, min(r0 + i, to - 1));
  }
}
// ... of [lo, hi) but for the whole tiles
template <typename T>
__device__ __forceinline__ void find_beside(const T* base, int64_t token, const Span& whole, int lo, int hi, int D, Span& at) {
  find_not_finite<T>(base, token, lo, whole.lo, D, at);
  find_not_finite<T>(base, token, whole.hi, hi, D, at);
}
constexpr Span kNowhere = {INT32_MAX, -1};

// Rows are formed again four at a time by matrix instructions of 4 x 4 in 16 blocks, fp32 sums, whose blocks do not mix: a score is of one row and one key
// alone, and what four rows of a sum take from a row of the other axis is left out, or added row by row, where not all of them see it.
constexpr int kAgain = 4;

// ---- of four rows: lanes hold elements lane + 64 c of their sums, and which of them are NaN where they are stored
struct Sums {
  f32x4 sum[kLaneCols];
  int lane, spoilt;  // bit 4 c + u
  template <typename E>
  __device__ __forceinline__ void find(int u, const E* stored, int D) {
#pragma unroll
    for (int c = 0; c < kLaneCols; ++c) {
      const float x = lane + 64 * c < D ? load_as_f32<E>(stored + lane + 64 * c) : 0.0f;
      spoilt |= x != x ? 1 << (4 * c + u) : 0;
    }
    spoilt = opaque(spoilt);
  }
  __device__ __forceinline__ void clear(int lane_) {
    lane = lane_, spoilt = 0;
#pragma unroll
    for (int c = 0; c < kLaneCols; ++c) sum[c] = f32x4{0, 0, 0, 0};
  }
  // an element that may still come out as a number
  __device__ __forceinline__ bool open() const {
    bool any = false;
#pragma unroll
    for (int c = 0; c < kLaneCols; ++c)
#pragma unroll
      for (int u = 0; u < kAgain; ++u) any |= (spoilt >> (4 * c + u) & 1) && sum[c][u] == sum[c][u];
    return __any(any);
  }
  template <typename Store>
  __device__ __forceinline__ void put(int u, Store store) const {
#pragma unroll
    for (int c = 0; c < kLaneCols; ++c)
      if (spoilt >> (4 * c + u) & 1) store(lane + 64 * c, sum[c][u]);
  }
};

// The next four of a wave's rows to be formed again: `at` says where values that are not finite lie in its masked tiles, and rows that see all of those
// keep what they have.  Lane i holds [from, to), what row row0 + i sees.
struct Four {
  int row0, lanes;     // the rows' lanes, six bits each from bit 8 u on, and a bit for those that keep what they have
  int lo, hi;          // lane i: what row i sees of [all_lo, all_hi) (held by the lanes: there are not as many scalar registers)
  int first, last;     // what any of them sees
  int i;               // lane % 4
  __device__ __forceinline__ void take(uint32_t& again, int lane_, int row0_, int from, int to, int all_lo, int all_hi, const Span& at) {
    i = lane_ & 3, row0 = row0_, lo = max(from, all_lo), hi = min(to, all_hi);
    lanes = 0, first = INT32_MAX, last = 0;
#pragma unroll
    for (int u = 0; u < kAgain; ++u) {
      const bool have = again != 0;
      const int l = have ? __builtin_ctz(again) : lanes & 63;
      again &= again - 1;
      const bool keeps = !have || (at.lo >= __builtin_amdgcn_readlane(from, l) && at.hi < __builtin_amdgcn_readlane(to, l));
      lanes |= (l | (keeps ? 64 : 0)) << 8 * u;
      const int a = __builtin_amdgcn_readlane(lo, l), b = __builtin_amdgcn_readlane(hi, l);
      if (!keeps && a < b) first = min(first, a), last = max(last, b);  // (a row whose keys all lie in other shares sees nothing here: its sum is 0)
    }
  }
  __device__ __forceinline__ int lane(int u) const { return lanes >> 8 * u & 63; }
  __device__ __forceinline__ int row(int u) const { return row0 + lane(u); }
  __device__ __forceinline__ bool keeps(int u) const { return lanes >> (8 * u + 6) & 1; }
  __device__ __forceinline__ bool sees(int u, int r) const {
    return !keeps(u) && __builtin_amdgcn_readlane(lo, lane(u)) <= r && r < __builtin_amdgcn_readlane(hi, lane(u));
  }
  // what lanes hold per row: that of row lane % 4
  __device__ __forceinline__ int my_lane() const { return lanes >> 8 * i & 63; }
  __device__ __forceinline__ int my_row() const { return row0 + my_lane(); }
  __device__ __forceinline__ float of_my_row(float v) const { return __shfl(v, my_lane(), kWave); }
  __device__ __forceinline__ int of_my_row(int v) const { return __shfl(v, my_lane(), kWave); }
};

// s[i] = a . b of the row a of lane 4 (lane / 4) + i and the lane's own row b, which lanes lane % 4 share
template <typename T>
__device__ __forceinline__ f32x4 four_dots(const T* a, const T* b, int D) {
  f32x4 s = {0, 0, 0, 0};
  if constexpr (sizeof(T) == 2) {  // (rows of whole 16 bytes that start there)
    auto eight = [&](const u32x4& x, const u32x4& y) {
      s = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(s16x4, u32x2{x[0], x[1]}), __builtin_bit_cast(s16x4, u32x2{y[0], y[1]}), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(s16x4, u32x2{x[2], x[3]}), __builtin_bit_cast(s16x4, u32x2{y[2], y[3]}), s, 0, 0, 0);
    };
    const u32x4 *x = reinterpret_cast<const u32x4*>(a), *y = reinterpret_cast<const u32x4*>(b);
    int n = D / 8;
    for (; n >= 4; n -= 4, x += 4, y += 4) {
      const u32x4 x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3], y0 = y[0], y1 = y[1], y2 = y[2], y3 = y[3];
      eight(x0, y0), eight(x1, y1), eight(x2, y2), eight(x3, y3);
    }
    for (; n > 0; --n) eight(*x++, *y++);
  } else {
    int d = 0;
    for (; d + 8 <= D; d += 8)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = __builtin_amdgcn_mfma_f32_4x4x1f32(a[d + i], b[d + i], s, 0, 0, 0);
    for (; d < D; ++d) s = __builtin_amdgcn_mfma_f32_4x4x1f32(a[d], b[d], s, 0, 0, 0);
  }
  return s;
}

// Adds w a of 16 rows a from `first` on that lie `token` apart: lane 4 b + u holds in w[i] the weight of row 4 b + i of 64 for the sum u; these are rows 16 PART on
template <typename T, int PART>
__device__ __forceinline__ void add_16(Sums& x, const f32x4& w, const Four& rows, const T* a, int64_t token, int first, int n, int D) {
  if (n <= 0) return;
  bool all = n >= 16;
#pragma unroll
  for (int u = 0; u < kAgain; ++u) all &= rows.keeps(u) || (rows.sees(u, first) && rows.sees(u, first + 15));  // (a sum that is not kept may take anything)
#pragma unroll
  for (int c = 0; c < kLaneCols; ++c) {
    if (64 * c >= D) break;
    const T* at = a + min(x.lane + 64 * c, D - 1);
    if (all) {
      T v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = at[i * token];
      auto block = [&](auto which) {
        constexpr int B = decltype(which)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (block 4 PART + B of the weights to all of them)
          x.sum[c] = __builtin_amdgcn_mfma_f32_4x4x1f32(w[i], load_as_f32<T>(&v[4 * B + i]), x.sum[c], 4, 4 * PART + B, 0);
      };
      block(std::integral_constant<int, 0>{});
      block(std::integral_constant<int, 1>{});
      block(std::integral_constant<int, 2>{});
      block(std::integral_constant<int, 3>{});
    } else {
      for (int i = 0; i < min(n, 16); ++i) {
        const float v = load_as_f32<T>(at + i * token), wi = (i & 2) ? ((i & 1) ? w[3] : w[2]) : ((i & 1) ? w[1] : w[0]);
#pragma unroll
        for (int u = 0; u < kAgain; ++u)
          if (rows.sees(u, first + i))
            x.sum[c][u] = fmaf(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wi), 16 * PART + (i & 12) + u)), v, x.sum[c][u]);
      }
    }
  }
}
// ... of n rows, up to 64
template <typename T>
__device__ __forceinline__ void add_rows(Sums& x, const f32x4& w, const Four& rows, const T* a, int64_t token, int first, int n, int D) {
  add_16<T, 0>(x, w, rows, a, token, first, n, D);
  add_16<T, 1>(x, w, rows, a + 16 * token, token, first + 16, n - 16, D);
  add_16<T, 2>(x, w, rows, a + 32 * token, token, first + 32, n - 32, D);
  add_16<T, 3>(x, w, rows, a + 48 * token, token, first + 48, n - 48, D);
}

// A wave's spoilt results over the keys of [all_lo, all_hi), by the rows' statistics, the last keys first; or with DQ its dq.  Lane i: of row row0 + i
template <typename T, bool DQ>
__device__ __forceinline__ void rows_again(const AttnArgs& p0, int h, int row0, uint32_t again, int start, float lse, float delta, int all_lo, int all_hi,
                                           const Span& whole, int share) {
  const int lane = lane_anew(), g = h / p0.group;
  Span at = kNowhere;
  if constexpr (DQ) find_beside(row_at<T>(p0.k, p0.k_token, p0.k_head, 0, g), p0.k_token, whole, all_lo, all_hi, p0.D, at);
  else find_beside(row_at<T>(p0.v, p0.v_token, p0.v_head, 0, g), p0.v_token, whole, all_lo, all_hi, p0.D, at);
  while (again) {
    const AttnArgs& p = late_arguments();  // (anew, rather than held in scalar registers over the loops)
    Four rows;
    rows.take(again, lane, row0, start, row0 + lane + 1, all_lo, all_hi, at);
    float* parts = (DQ ? p.dq_part : p.out_part) + static_cast<int64_t>(share) * p.T * p.H * p.D_out;
    T* stored = static_cast<T*>(DQ ? p.dq : p.out);
    Sums x;
    x.clear(lane);
#pragma unroll
    for (int u = 0; u < kAgain; ++u) {
      const int64_t dense = (static_cast<int64_t>(rows.row(u)) * p.H + h) * p.D_out;
      if (p.share_bits) x.find(u, parts + dense, rows.keeps(u) ? 0 : p.D_out);
      else x.find(u, stored + dense, rows.keeps(u) ? 0 : p.D_out);
    }
    const int64_t my_row = rows.my_row();
    const T *q = row_at<T>(p.q, p.q_token, p.q_head, my_row, h), *dout = DQ ? static_cast<const T*>(p.dout) + (my_row * p.H + h) * p.D : nullptr;
    const float my_lse = rows.of_my_row(lse), my_delta = DQ ? rows.of_my_row(delta) : 0.0f;
    // (a row that sees one key: its weight is 1, whatever its score)
    const bool several = rows.of_my_row(start) < my_row;
    for (int to = rows.last; rows.first < to && x.open(); to -= kWave) {
      const int j0 = max(to - kWave, rows.first), j = min(j0 + lane, to - 1);
      const T *k = row_at<T>(p.k, p.k_token, p.k_head, j, g), *v = row_at<T>(p.v, p.v_token, p.v_head, j, g);
      f32x4 w = four_dots<T>(k, q, p.D);
      if constexpr (DQ) {
        const f32x4 dp = four_dots<T>(v, dout, p.D);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = several ? exp2_f32(fmaf(w[i], p.c, -my_lse)) * (dp[i] - my_delta) : 0.0f;
        add_rows<T>(x, w, rows, row_at<T>(p.k, p.k_token, p.k_head, j0, g), p.k_token, j0, to - j0, p.D);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = exp2_f32(fmaf(w[i], p.c, -my_lse));
        add_rows<T>(x, w, rows, row_at<T>(p.v, p.v_token, p.v_head, j0, g), p.v_token, j0, to - j0, p.D);
      }
    }
#pragma unroll
    for (int u = 0; u < kAgain; ++u) {
      const int64_t dense = (static_cast<int64_t>(rows.row(u)) * p.H + h) * p.D_out;
      x.put(u, [&](int d, float sum) {
        if (DQ) sum *= p.scale;
        if (p.share_bits) parts[dense + d] = sum;
        else if (DQ) store_from_f32<T>(stored + dense + d, sum);
        else store_result<T>(p, dense + d, sum);
      });
    }
  }
}

// ... and dk and dv of a wave's keys over the rows of [all_lo, all_hi) of the query heads [h0, h1), into the part `split` where there are parts, the
// first rows first; delta is kept times `sign`
template <typename T>
__device__ __forceinline__ void keys_again(const AttnArgs& p0, int g, int key0, uint32_t again, int start, int end, int h0, int h1, int all_lo, int all_hi,
                                           const Span& whole, int split, float sign) {
  const int lane = lane_anew();
  const int64_t dense_token = static_cast<int64_t>(p0.H) * p0.D;
  Span at = kNowhere;
#pragma clang loop unroll(disable)
  for (int i = 2 * h0; i < 2 * h1; ++i) {
    const AttnArgs& p = late_arguments();
    if (i & 1) find_beside(static_cast<const T*>(p.dout) + (i >> 1) * p.D, dense_token, whole, all_lo, all_hi, p.D, at);
    else find_beside(row_at<T>(p.q, p.q_token, p.q_head, 0, i >> 1), p.q_token, whole, all_lo, all_hi, p.D, at);
  }
#pragma clang loop unroll(disable)
  for (int to_dk = 0; to_dk < 2; ++to_dk) {
    for (uint32_t left = again; left;) {
      const AttnArgs& p = late_arguments();
      Four keys;
      keys.take(left, lane, key0, key0 + lane, end, all_lo, all_hi, at);
      // where the gradient of key u lies, as a part or in the storage type
      auto with_stored = [&](int u, auto f) {
        const AttnArgs& p = late_arguments();
        const int64_t dense = (static_cast<int64_t>(keys.row(u)) * p.G + g) * p.D_out;
        if (p.splits > 1) f((to_dk ? p.dk_part : p.dv_part) + static_cast<int64_t>(split) * p.T * p.G * p.D_out + dense, p);
        else f(static_cast<T*>(to_dk ? p.dk : p.dv) + dense, p);
      };
      Sums x;
      x.clear(lane);
#pragma unroll
      for (int u = 0; u < kAgain; ++u) with_stored(u, [&](auto* stored, const AttnArgs& p) { x.find(u, stored, keys.keeps(u) ? 0 : p.D_out); });
      const int64_t my_key = keys.my_row();
      const T *k = row_at<T>(p.k, p.k_token, p.k_head, my_key, g), *v = row_at<T>(p.v, p.v_token, p.v_head, my_key, g);
      const int my_start = keys.of_my_row(start);
      for (int h = h0; h < h1; ++h) {
        const T *q = row_at<T>(p.q, p.q_token, p.q_head, 0, h), *dout = static_cast<const T*>(p.dout) + h * p.D;
        const float *lse = p.lse + static_cast<int64_t>(h) * p.T, *delta = p.delta + static_cast<int64_t>(h) * p.T;
        for (int r0 = keys.first; r0 < keys.last && x.open(); r0 += kWave) {
          const int n = min(keys.last - r0, kWave);
          const int64_t r = r0 + min(lane, n - 1);
          f32x4 w = four_dots<T>(q + r * p.q_token, k, p.D);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = exp2_f32(fmaf(w[i], p.c, -lse[r0 + min((lane & ~3) + i, n - 1)]));
          if (to_dk) {
            const f32x4 dp = four_dots<T>(dout + r * dense_token, v, p.D);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int ri = r0 + min((lane & ~3) + i, n - 1);
              w[i] = my_start < ri ? w[i] * (dp[i] - sign * delta[ri]) : 0.0f;
            }
          }
          const int64_t token = to_dk ? p.q_token : dense_token;
          add_rows<T>(x, w, keys, (to_dk ? q : dout) + r0 * token, token, r0, n, p.D);
        }
      }
#pragma unroll
      for (int u = 0; u < kAgain; ++u)
        with_stored(u, [&](auto* stored, const AttnArgs& p) {
          x.put(u, [&](int d, float sum) { store_from_f32(stored + d, to_dk ? sum * p.scale : sum); });
        });
    }
  }
}

// ---- order of the tiles ---------------------------------------------------------------------------------
// A tile's work is as long as the other axis that its rows see.  Of one sequence the last rows see the most; of several nothing about
// it is known without cu_seqlens, and a heavy tile that starts last ends long after the others.  Where there are more
// workgroups than the card holds at once and sequences are long on average (entries of cu_seqlens, empty ones among them), one small kernel (5 us) sorts
// the tiles by their work first: the backward from 512 rows a sequence on, the forward, whose tiles take a third of the time, from 1024.  us not sorted -> sorted,
// even lengths; uneven ones (split at random), on one machine:
//   forward   8192 rows, 32/4 heads of 128   2048 a sequence 185 -> 184; 205 -> 206   1024 99 -> 101; 134 -> 133    512 69 -> 76; 112 -> 113
//             8192, 16/16 of 64                         73 -> 57; 99 -> 107           42 -> 37; 59 -> 60            28 -> 29; 50 -> 55
//             fp32 4096, 8/2 of 64                      113 -> 112; 112 -> 117        80 -> 74; 92 -> 93            56 -> 54; 64 -> 63
//   forward   8192 rows, 32/4 heads of 128   2048 781 -> 716; 1043 -> 1056            512 359 -> 364; 587 -> 560    256 290 -> 320; 457 -> 444
//   and       8192, 16/16 of 64                   257 -> 229; 383 -> 395                  122 -> 119; 215 -> 202         96 -> 105; 169 -> 165
//   backward  fp32 4096, 8/2 of 64                465 -> 456; 473 -> 476                  217 -> 194; 261 -> 234         156 -> 146; 227 -> 213
constexpr int kHeldAtOnce = 512;             // workgroups: two a CU
constexpr int kLongForward = 1024, kLongBackward = 512;  // rows a sequence: below, a tile's work differs by less than the sorting costs
inline bool sorted_tiles(int64_t sequences, int64_t T, int64_t tiles, int64_t heads, int rows_each) {
  return sequences > 1 && T >= rows_each * sequences && tiles * heads > kHeldAtOnce / 2;
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
