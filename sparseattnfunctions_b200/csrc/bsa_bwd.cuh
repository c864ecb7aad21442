// bsa_bwd.cuh -- what the two gradient kernels of block-sparse attention share:
// the workspace layout, and the parameters of the preparation launch.
//
// Mathematics (c = sm_scale, over the listed blocks):
//   p_ij  = exp(c q_i.k_j - lse_i)        dp_ij = do_i . v_j
//   delta_i = do_i . o_i                  ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij do_i    dq_i = c sum_j ds_ij k_j    dk_j = c sum_i ds_ij q_i
// p is recomputed from the log-sum-exp; nothing of size Sq x Sk is stored.
// Every output tile is owned by one work item, which walks its own list of
// blocks in ascending order: a query tile's key blocks (dq) or a key tile's
// query blocks (dk, dv).  The products s and dp are formed in both walks
// (7 matrix products instead of 5; the 16-bit kernel runs an eighth, of what
// rounding takes off dq's ds), and in return no gradient is accumulated by
// atomics: equal inputs give equal bits.
#pragma once

#include "saf_common.cuh"

namespace saf {

// Workspace of one call.  A line is the tile of mask rows (dq) or mask columns
// (dk, dv) of one work item: one mask block, or two where 64-token blocks fill
// a 128-token tile of the 16-bit kernel.  Lists: [BH, lines, cap] entries
// block index | live halves of the line << 14, ascending; counts [BH, lines].
struct BwdWorkspace {
  float* stat_lse;    // [BH, Sp]: -lse (16-bit kernel: in log2 units, plus p's scale), -inf where nothing is seen
  float* stat_delta;  // [BH, Sp]: -delta
  uint16_t* list_q;   // dq lines -> key blocks
  uint16_t* list_k;   // dk / dv lines -> query blocks
  int32_t* count_q;
  int32_t* count_k;
  // 16-bit kernel only: work items by length (longest class first) and the
  // counters, zeroed before the preparation
  uint2* items;          // [kClasses][item_cap]: (1 << 31 for dk / dv) | head * lines + line, part (see PartOf)
  int32_t* class_count;  // [kClasses]
  int32_t* next;         // the next item to take
  int item_cap;
  // with few heads, long lists are cut into parts whose fp32 sums [128, 64]
  // (dk or dq, then dv) meet in bwd_merge_kernel; part_cap 0: no list is cut
  int part_cap;          // parts that fit (16-bit: part is [part_cap][2][128 x 64])
  int32_t* parts_used;
  int32_t* split_count;  // lines cut
  uint2* split;          // [part_cap / 2]: the line as in items, its first part and their number
  // f16 only: what a row's largest |do| puts into dS's exponent, the largest
  // |do| of each 64 rows, and the largest finite |v| of each head
  float* stat_exp;  // [BH, Sp]
  float* amax;      // [BH, Sp / 64]
  uint32_t* vmax;   // [BH], bits of the float; zeroed with the counters
  float* part;  // partial sums
  // fp32 kernel only: CTAs that share a tile, and the tiles' counts of finished ones
  int chunks;
  int* part_count;
  int lines_q, lines_k, cap_q, cap_k;
  int64_t Sp;  // Sq rounded up to 128
  size_t bytes;
};

// f16: dS times 2^4 (P's factor) and 2^e stays below 2^15 whatever the signs:
// |do . v - delta| <= 128 |do| |v| (o is a mean of v), each below twice its
// power of two, so e = 2 - ilogb(largest |do|) - ilogb(largest |v|).  The two
// parts of it; 0 where all are zero or not finite.
__device__ __forceinline__ int f16_exponent(float a) { return a > 0.f && a <= 65504.f ? ilogbf(a) : 0; }
__device__ __forceinline__ int f16_ds_exponent_do(float a) { return -f16_exponent(a); }
__device__ __forceinline__ int f16_ds_exponent_v(float a) { return 2 - f16_exponent(a); }
// 2^e, |e| <= 126
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

// Length classes of the work items: class 15 - floor(log2(blocks)), so that
// the longest lists start first and the short ones fill the last wave.
constexpr int kClasses = 16;

// Second word of an item: place in `part` | number of the part << 16 | parts << 24
// (1 part: the line is whole).
struct PartOf {
  int slot, number, parts;
};
__host__ __device__ inline uint32_t pack_part(int slot, int number, int parts) {
  return static_cast<uint32_t>(slot) | static_cast<uint32_t>(number) << 16 | static_cast<uint32_t>(parts) << 24;
}
__host__ __device__ inline PartOf unpack_part(uint32_t x) {
  return PartOf{static_cast<int>(x & 0xffffu), static_cast<int>(x >> 16 & 0xffu), static_cast<int>(x >> 24)};
}

}  // namespace saf
