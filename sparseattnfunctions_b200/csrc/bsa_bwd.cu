// bsa_bwd.cu -- gradient of block-sparse attention: entry points, the
// preparation launch (row statistics, per-tile block lists, work items) and
// the fp32 gradient kernel on the CUDA cores (16 bits: bsa_bwd_sm100.cu).  Formulas and work split: bsa_bwd.cuh.
#include "bsa_bwd.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace saf {

float bwd_f16_p_log2_scale();
int32_t bsa_bwd_sm100(const saf_tensor4* dout, const saf_tensor4* q, const saf_tensor4* k, const saf_tensor4* v,
                      const saf_tensor4* dq, const saf_tensor4* dk, const saf_tensor4* dv, int bm, int bn,
                      float sm_scale, const BwdWorkspace& w, cudaStream_t stream);

namespace {

constexpr int kT = 64;            // sub-tile edge of the CUDA-core kernel
constexpr int kSimtThreads = 256;
constexpr int kGroup = 32;        // mask lines one list block handles
constexpr int kRowChunk = 128;    // rows one statistics block handles
constexpr int kMaxBlocks = 16384; // 14-bit block indexes in the lists
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCounters = kClasses + 3;  // class counts, next item, parts, cut lines
// A line is cut when it holds more than 1.5 times kMinPart tiles of 128 x 128,
// and than 1.5 times an SM's share of the work (estimated from its own head's
// listed blocks); a part holds about that many.  Parts number at most 1.67
// times the tiles over the share, times up to 4 where 64-token blocks fill
// tiles sparsely: under kPartCap.
constexpr int kMinPart = 12, kPartCap = 1024, kMaxParts = 32;

// Mask lines that share a tile: 64-token blocks pair up under the 16-bit kernel.
int merge_of(int32_t dtype, int block) { return dtype != SAF_F32 && block == 64 ? 2 : 1; }

int simt_chunks(int64_t tiles);

BwdWorkspace layout(const saf_tensor4* q, const saf_tensor4* k, int bm, int bn, uint8_t* base) {
  BwdWorkspace w{};
  const int64_t BH = q->B * q->H;
  const int64_t nbq = (q->S + bm - 1) / bm, nbk = (k->S + bn - 1) / bn;
  const int mq = merge_of(q->dtype, bm), mk = merge_of(q->dtype, bn);
  w.Sp = (q->S + 127) / 128 * 128;
  w.lines_q = static_cast<int>((nbq + mq - 1) / mq);
  w.lines_k = static_cast<int>((nbk + mk - 1) / mk);
  w.cap_q = static_cast<int>((nbk + 7) / 8 * 8);
  w.cap_k = static_cast<int>((nbq + 7) / 8 * 8);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* ptr = base + at;
    at = (at + bytes + 255) / 256 * 256;
    return ptr;
  };
  w.stat_lse = reinterpret_cast<float*>(take(static_cast<size_t>(BH * w.Sp) * 4));
  w.stat_delta = reinterpret_cast<float*>(take(static_cast<size_t>(BH * w.Sp) * 4));
  w.list_q = reinterpret_cast<uint16_t*>(take(static_cast<size_t>(BH * w.lines_q) * w.cap_q * 2));
  w.list_k = reinterpret_cast<uint16_t*>(take(static_cast<size_t>(BH * w.lines_k) * w.cap_k * 2));
  w.count_q = reinterpret_cast<int32_t*>(take(static_cast<size_t>(BH * w.lines_q) * 4));
  w.count_k = reinterpret_cast<int32_t*>(take(static_cast<size_t>(BH * w.lines_k) * 4));
  if (q->dtype != SAF_F32) {
    // Cutting pays where one list outlasts an SM's share of the whole.  Whole
    // and cut lists, a tenth of the 128-blocks and dense text, us: one head of
    // 17776 tokens 229 and 94; two of 2500, 4000, 17776, 33976 tokens 43 and 41,
    // 61 and 45, 225 and 139, 423 and 441; three of 4000, 8000, 17776, 33976
    // tokens 69 and 56, 114 and 79, 225 and 235, 475 and 487; four of 17776
    // 225 and 236.
    const int64_t longest = (q->S > k->S ? q->S : k->S) / 128;
    w.part_cap = BH <= 3 && 2 * longest > 3 * kMinPart ? kPartCap : 0;
    w.item_cap = static_cast<int>(BH * (w.lines_q + w.lines_k)) + w.part_cap;
    w.items = reinterpret_cast<uint2*>(take(static_cast<size_t>(w.item_cap) * kClasses * 8));
    const int64_t vmax = q->dtype == SAF_F16 ? BH : 0;
    w.class_count = reinterpret_cast<int32_t*>(take(static_cast<size_t>(kCounters + vmax) * 4));
    w.vmax = reinterpret_cast<uint32_t*>(w.class_count + kCounters);
    w.next = w.class_count + kClasses;
    w.parts_used = w.next + 1;
    w.split_count = w.next + 2;
    if (w.part_cap > 0) {
      w.part = reinterpret_cast<float*>(take(static_cast<size_t>(w.part_cap) * 2 * 128 * 64 * 4));
      w.split = reinterpret_cast<uint2*>(take(static_cast<size_t>(w.part_cap / 2) * 8));
    }
    if (q->dtype == SAF_F16) {
      w.stat_exp = reinterpret_cast<float*>(take(static_cast<size_t>(BH * w.Sp) * 4));
      w.amax = reinterpret_cast<float*>(take(static_cast<size_t>(BH * (w.Sp / 64)) * 4));
    }
  }
  if (q->dtype == SAF_F32) {
    const int64_t tk = (k->S + kT - 1) / kT, tq = (q->S + kT - 1) / kT;
    w.chunks = simt_chunks(BH * (tk + tq));
    if (w.chunks > 1) {
      w.part = reinterpret_cast<float*>(take(static_cast<size_t>(BH * (2 * tk + tq)) * w.chunks * kT * q->D * 4));
      w.part_count = reinterpret_cast<int*>(take(static_cast<size_t>(BH * (tk + tq)) * 4));
    }
  }
  w.bytes = at;
  return w;
}

// ---------------------------------------------------------------------------
// Preparation: one launch of list blocks and statistics blocks, so that the
// short chains of the lists hide behind the statistics' reading of out and
// dout.  Bound by HBM at large sizes (60 heads of 17776 tokens, 16 bits: 273 MB
// in 62 us, 4.4 TB/s), by a chain of dependent loads at small ones (4 us).
// ---------------------------------------------------------------------------

struct PrepParams {
  const void* out;
  const void* dout;
  const void* v;
  int64_t o_sb, o_sh, o_ss, d_sb, d_sh, d_ss, v_sb, v_sh, v_ss;
  int H, Sq, Sk, D;
  const float* lse;
  int64_t lse_stride;  // per head
  float lse_factor, lse_shift;  // stat_lse = lse_shift - lse_factor * lse
  int items;                    // 1: fill the work items
  int nbq, nbk, bm, bn, merge_q, merge_k;
  int groups_q, groups_k;
  const int32_t* row_ptr;
  const int32_t* col_idx;
  int64_t col_capacity;
  BwdWorkspace w;
  unsigned int* status;
};

// The lists of 32 mask rows or columns of head g: a bitmap of the live blocks
// of each line, filled from the listed entries and read back ascending.
// A line with an entry outside the mask sets the bad-index flag and skips it.
__device__ void build_lists(const PrepParams& p, int g, int group, bool columns) {
  extern __shared__ uint32_t sm[];
  __shared__ int cls_n[kClasses], cls_at[kClasses], my_cls[kGroup], my_pos[kGroup];
  __shared__ uint32_t my_part[kGroup];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int other = columns ? p.nbq : p.nbk, words = (other + 31) >> 5;
  uint32_t* bits = sm;                                       // [32][words]
  int32_t* rp = reinterpret_cast<int32_t*>(sm + kGroup * words);  // [rows + 1]
  const int line0 = group * kGroup;
  const int row0 = columns ? 0 : line0;
  const int rows = columns ? p.nbq : min(kGroup, p.nbq - line0);
  for (int i = tid; i < kGroup * words; i += blockDim.x) bits[i] = 0u;
  if (tid < kClasses) cls_n[tid] = 0;
  const int32_t* src = p.row_ptr + static_cast<int64_t>(g) * (p.nbq + 1) + row0;
  for (int i = tid; i <= rows; i += blockDim.x) {
    const int32_t x = src[i];
    rp[i] = x < 0 ? 0 : (static_cast<int64_t>(x) > p.col_capacity ? static_cast<int32_t>(p.col_capacity) : x);
  }
  __syncthreads();
  // a warp takes four rows at a time, a lane every 32nd entry of each
  for (int r0 = warp * 4; r0 < rows; r0 += 32) {
    int at[4], end[4], most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] = r0 + i < rows ? rp[r0 + i] : 0;
      end[i] = r0 + i < rows ? rp[r0 + i + 1] : 0;
      most = max(most, end[i] - at[i]);
    }
    for (int k = lane; k - lane < most; k += 32) {
      int c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = k < end[i] - at[i] ? p.col_idx[at[i] + k] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k >= end[i] - at[i]) continue;
        if (c[i] < 0 || c[i] >= p.nbk) {
          atomicOr(p.status, SAF_DEV_BADINDEX);
          continue;
        }
        const int line = columns ? c[i] - line0 : r0 + i, bit = columns ? row0 + r0 + i : c[i];
        if (line >= 0 && line < kGroup) atomicOr(&bits[line * words + (bit >> 5)], 1u << (bit & 31));
      }
    }
  }
  __syncthreads();
  const int merge = columns ? p.merge_k : p.merge_q;
  const int lines = columns ? p.w.lines_k : p.w.lines_q, cap = columns ? p.w.cap_k : p.w.cap_q;
  uint16_t* list = columns ? p.w.list_k : p.w.list_q;
  int32_t* count = columns ? p.w.count_k : p.w.count_q;
  for (int t = warp; t < kGroup / merge; t += blockDim.x >> 5) {
    const int tile = line0 / merge + t;
    if (tile >= lines) break;
    const uint32_t* ba = bits + t * merge * words;
    const uint32_t* bb = ba + (merge - 1) * words;
    uint16_t* dst = list + (static_cast<int64_t>(g) * lines + tile) * cap;
    int n = 0;
    for (int w0 = 0; w0 < words; w0 += 32) {
      const int w = w0 + lane;
      const uint32_t a = w < words ? ba[w] : 0u, b = w < words ? bb[w] : 0u;
      uint32_t u = a | b;
      int incl = __popc(u);
      const int cnt = incl;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
      }
      int pos = n + incl - cnt;
      while (u != 0u) {
        const int bit = __ffs(u) - 1;
        u &= u - 1u;
        const uint32_t half = ((a >> bit) & 1u) | (((b >> bit) & 1u) << 1);
        dst[pos++] = static_cast<uint16_t>((w * 32 + bit) | (half << 14));
      }
      n += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      const uint32_t id = static_cast<uint32_t>(g * lines + tile);
      count[id] = n;
      if (p.items) {
        const int other_block = columns ? p.bm : p.bn;
        const int tiles = other_block == 64 ? (n + 1) / 2 : n;
        int parts = 1, slot = 0;
        if (p.w.part_cap > 0) {
          const int64_t entries = p.row_ptr[static_cast<int64_t>(g) * (p.nbq + 1) + p.nbq] -
                                  p.row_ptr[static_cast<int64_t>(g) * (p.nbq + 1)];
          const int64_t work = 2 * entries * (p.bm * p.bn) / (128 * 128) * gridDim.x;
          const int64_t share = max(static_cast<int64_t>(kMinPart), (work + kPlannedSms - 1) / kPlannedSms);
          if (2 * static_cast<int64_t>(tiles) > 3 * share) {
            parts = static_cast<int>(min(static_cast<int64_t>(kMaxParts), (tiles + share - 1) / share));
            slot = atomicAdd(p.w.parts_used, parts);
            if (slot + parts > p.w.part_cap) parts = 1, slot = 0;
          }
          if (parts > 1)
            p.w.split[atomicAdd(p.w.split_count, 1)] =
                make_uint2((columns ? 0x80000000u : 0u) | id, pack_part(slot, 0, parts));
        }
        const int len = (tiles + parts - 1) / parts;
        const int cls = kClasses - 1 - (len > 0 ? 31 - __clz(len) : 0);
        my_cls[t] = cls;
        my_part[t] = pack_part(slot, 0, parts);
        my_pos[t] = atomicAdd(&cls_n[cls], parts);
      }
    }
  }
  if (!p.items) return;
  // this block's items, class by class, behind those of the blocks before it
  __syncthreads();
  if (tid < kClasses && cls_n[tid] > 0) cls_at[tid] = atomicAdd(&p.w.class_count[tid], cls_n[tid]);
  __syncthreads();
  const int tile = line0 / merge + tid;
  if (tid < kGroup / merge && tile < lines) {
    uint2* at = p.w.items + static_cast<int64_t>(my_cls[tid]) * p.w.item_cap + cls_at[my_cls[tid]] + my_pos[tid];
    const PartOf part = unpack_part(my_part[tid]);
    for (int i = 0; i < part.parts; ++i)
      at[i] = make_uint2((columns ? 0x80000000u : 0u) | static_cast<uint32_t>(g * lines + tile),
                         pack_part(part.slot + i, i, part.parts));
  }
}

__device__ __forceinline__ float2 unpack2(uint32_t x, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t x, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// -delta and the negative log-sum-exp of 128 rows of head g.  A row that sees
// no key (lse -inf) and the rows that pad the last tile get -inf, so that
// every exp(s - lse) of theirs is 0.  f16: also what the rows' and the two
// 64-row blocks' largest |do| ask for.
template <typename T>
__device__ void row_stats(const PrepParams& p, int g, int chunk) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = g / p.H, h = g % p.H;
  const T* o = static_cast<const T*>(p.out) + b * p.o_sb + h * p.o_sh;
  const T* d = static_cast<const T*>(p.dout) + b * p.d_sb + h * p.d_sh;
  const int64_t base = static_cast<int64_t>(g) * p.w.Sp;
  auto store = [&](int row, float delta) {
    const float l = row < p.Sq ? p.lse[g * p.lse_stride + row] : -INFINITY;
    p.w.stat_lse[base + row] = l == -INFINITY ? -INFINITY : p.lse_shift - l * p.lse_factor;
    p.w.stat_delta[base + row] = l == -INFINITY ? 0.f : -delta;
  };
  if constexpr (sizeof(T) == 2) {  // D = 64: 8 lanes of 16 bytes a row
    const int sub = lane & 7;
    constexpr bool kMax = std::is_same<T, __half>::value;
    float amax[2] = {0.f, 0.f};  // of the chunk's two 64-row blocks
    constexpr int kRows = kRowChunk / 32;  // a thread's rows, all in flight
    uint4 x[kRows], y[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = chunk * kRowChunk + i * 32 + warp * 4 + (lane >> 3);
      const bool in = row < p.Sq;
      x[i] = in ? *reinterpret_cast<const uint4*>(o + row * p.o_ss + sub * 8) : uint4{0, 0, 0, 0};
      y[i] = in ? *reinterpret_cast<const uint4*>(d + row * p.d_ss + sub * 8) : uint4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = chunk * kRowChunk + i * 32 + warp * 4 + (lane >> 3);
      float sum = 0.f, row_max = 0.f;
      const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 fx = unpack2(xs[e], static_cast<const T*>(nullptr));
        const float2 fy = unpack2(ys[e], static_cast<const T*>(nullptr));
        sum = fmaf(fx.x, fy.x, fmaf(fx.y, fy.y, sum));
        if constexpr (kMax) row_max = fmaxf(row_max, fmaxf(fabsf(fy.x), fabsf(fy.y)));
      }
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (sub == 0) store(row, sum);
      if constexpr (kMax) {
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) row_max = fmaxf(row_max, __shfl_xor_sync(0xffffffffu, row_max, off));
        if (sub == 0) p.w.stat_exp[base + row] = static_cast<float>(f16_ds_exponent_do(row_max));
        amax[i / 2] = fmaxf(amax[i / 2], row_max);
      }
    }
    if constexpr (kMax) {
      __shared__ float warp_max[2][8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 16; off > 4; off >>= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], off));
        if (lane == 0) warp_max[i][warp] = amax[i];
      }
      __syncthreads();
      if (threadIdx.x < 2) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, warp_max[threadIdx.x][i]);
        p.w.amax[g * (p.w.Sp / 64) + 2 * chunk + threadIdx.x] = m;
      }
    }
  } else {
    // a warp's 16 rows, four at a time in flight
    for (int r0 = warp; r0 < kRowChunk; r0 += 32) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int e = lane; e < p.D; e += 32)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = chunk * kRowChunk + r0 + 8 * i;
          if (row < p.Sq) sum[i] = fmaf(o[row * p.o_ss + e], d[row * p.d_ss + e], sum[i]);
        }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], off);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane == 0) store(chunk * kRowChunk + r0 + 8 * i, sum[i]);
    }
  }
}

// f16: the largest finite |v| of 128 rows of head g (an infinity decides nothing:
// what sees it is not finite anyway, and the others keep their scale).
__device__ void value_max(const PrepParams& p, int g, int chunk) {
  const __half* v = static_cast<const __half*>(p.v) + g / p.H * p.v_sb + g % p.H * p.v_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint4 x[kRowChunk / 32];
#pragma unroll
  for (int i = 0; i < kRowChunk / 32; ++i) {
    const int row = chunk * kRowChunk + i * 32 + warp * 4 + (lane >> 3);
    x[i] = row < p.Sk ? *reinterpret_cast<const uint4*>(v + row * p.v_ss + (lane & 7) * 8) : uint4{0, 0, 0, 0};
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kRowChunk / 32; ++i)
#pragma unroll
    for (const uint32_t w : {x[i].x, x[i].y, x[i].z, x[i].w}) {
      const float2 f = unpack2(w, static_cast<const __half*>(nullptr));
      const float a = fabsf(f.x), b = fabsf(f.y);
      m = fmaxf(m, fmaxf(a < INFINITY ? a : 0.f, b < INFINITY ? b : 0.f));
    }
  const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // non-negative floats order as integers
  if (lane == 0) atomicMax(p.w.vmax + g, most);
}

template <typename T>
__global__ void __launch_bounds__(256) bwd_prep_kernel(const PrepParams p) {
  const int g = blockIdx.x, x = blockIdx.y;  // every head's lists start before the statistics
  // the 16-bit gradient may set itself up once every block here has started
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (x < p.groups_k)
    build_lists(p, g, x, true);
  else if (x < p.groups_k + p.groups_q)
    build_lists(p, g, x - p.groups_k, false);
  else if (const int chunk = x - p.groups_k - p.groups_q; chunk < p.w.Sp / kRowChunk)
    row_stats<T>(p, g, chunk);
  else if constexpr (std::is_same<T, __half>::value)
    value_max(p, g, chunk - static_cast<int>(p.w.Sp / kRowChunk));
}

// ---------------------------------------------------------------------------
// CUDA-core gradient (fp32: the caller wants fp32 accuracy, which TF32 products
// do not have).  A CTA's two operand pairs lie row-major in shared memory and
// are read back in both orders; a thread owns 4 x 4 of a 64 x 64 sub-tile.
// Bound by shared-memory reads and issue (counters: LSU 55 %, issue 60 %): 2
// heads of 2048 tokens, a quarter of the 64-blocks, take 100 us.  Such
// sizes have fewer tiles than the GPU takes CTAs, so several CTAs share a
// tile's walk and the last one to finish adds their sums in a fixed order.
// Larger sizes run the seven products at 26 to 30 TFLOP/s of 72 (16 heads of
// 4096 tokens 2.4 ms); tiles of 8 x 4 a thread and half the threads left that
// as it is (2.36 ms) and cost the small sizes 10 %.
// ---------------------------------------------------------------------------

struct SimtBwdParams {
  const float *q, *k, *v, *dout;
  float *dq, *dk, *dv;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss, do_sb, do_sh, do_ss;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int H, Sq, Sk, bm, bn, tiles_k;
  float scale;
  bool vec;  // every row of q, k, v, dout starts at a multiple of 16 bytes
  int chunks, part_tiles;  // CTAs a tile; partial tiles a head (two a key tile, one a query tile)
  float* part;
  int* part_count;  // [BH, tiles]
  BwdWorkspace w;
};

// Rows [r0, r0 + 64) of two [S, D] views into dst1 and dst2 [64][D + 4], zeros
// past S; all of a thread's loads of a pass are in flight before its stores.
// vec: every row starts at a multiple of 16 bytes.
template <int D>
__device__ __forceinline__ void load_tiles(float* dst1, const float* src1, int64_t ss1, float* dst2, const float* src2,
                                           int64_t ss2, int r0, int S, bool vec) {
  if (vec) {
    constexpr int kPass = 4;
#pragma unroll
    for (int j0 = 0; j0 < kT * D / 4 / kSimtThreads; j0 += kPass) {
      float4 x[kPass], y[kPass];
#pragma unroll
      for (int j = 0; j < kPass; ++j) {
        const int i = threadIdx.x + (j0 + j) * kSimtThreads, r = i / (D / 4), d = i % (D / 4) * 4;
        const bool in = r0 + r < S;
        x[j] = in ? *reinterpret_cast<const float4*>(src1 + (r0 + r) * ss1 + d) : float4{0.f, 0.f, 0.f, 0.f};
        y[j] = in ? *reinterpret_cast<const float4*>(src2 + (r0 + r) * ss2 + d) : float4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = 0; j < kPass; ++j) {
        const int i = threadIdx.x + (j0 + j) * kSimtThreads, r = i / (D / 4), d = i % (D / 4) * 4;
        *reinterpret_cast<float4*>(dst1 + r * (D + 4) + d) = x[j];
        *reinterpret_cast<float4*>(dst2 + r * (D + 4) + d) = y[j];
      }
    }
  } else {
    for (int i = threadIdx.x; i < kT * D; i += kSimtThreads) {
      const int r = i / D, d = i % D;
      const bool in = r0 + r < S;
      dst1[r * (D + 4) + d] = in ? src1[(r0 + r) * ss1 + d] : 0.f;
      dst2[r * (D + 4) + d] = in ? src2[(r0 + r) * ss2 + d] : 0.f;
    }
  }
}

__device__ __forceinline__ float dot4(float4 a, float4 b, float c) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, c))));
}

template <int D>
constexpr int kSimtSmem = (4 * kT * (D + 4) + 2 * kT * (kT + 4) + 2 * kT) * 4;

// CTAs that share a tile's walk, sub-tile by sub-tile in turn: with few tiles
// one CTA a tile leaves the GPU idle behind the longest list.  Enough for eight
// CTAs an SM, at most 8; from 1184 tiles on there is no split.  Unsplit, two
// heads of 32 tiles each way at 2048 tokens took 200 us.  With enough for 4, 8,
// 12 an SM (at most 16): those and a dense column 146, 139, 145 us, eight heads
// 424, 378, 376, four heads of 4096 tokens in 128-blocks 727, 625, 592; all of
// 2 x 1000 tokens 108, 109, 128.
int simt_chunks(int64_t tiles) {
  const int64_t want = (8 * kPlannedSms + tiles - 1) / tiles;
  return static_cast<int>(want < 1 ? 1 : want > 8 ? 8 : want);
}

// p.chunks CTAs per 64 output rows: key rows (dk and dv) for tile < tiles_k,
// query rows (dq) after them.  The tile's own two operands (k, v or q, do)
// stay in shared memory; the walk brings the other two.  Thread (ty, tx) of a
// 16 x 16 grid forms the scores of walked rows ty + 16a against own rows
// tx + 16c, then owns output rows ty*4..+3, channels tx*4..+3 (twice at
// D = 128).  The partial sums of a split tile go to the workspace; the CTA
// that finishes last adds them in the order of the chunks.  Bound by
// shared-memory reads and the FMA pipe.
template <int D, bool kKeys>
__device__ void simt_tile(const SimtBwdParams& p, int g, int tile, int chunk) {
  constexpr int LD = D + 4, DC = D / 64;
  extern __shared__ float smf[];
  float* a1 = smf;                                // own k or q
  float* a2 = a1 + kT * LD;                       // own v or do
  float* b1 = a2 + kT * LD;                       // walked q or k
  float* b2 = b1 + kT * LD;                       // walked do or v
  float* ps = b2 + kT * LD;                       // [walked row][own row] p
  float* ds = ps + kT * (kT + 4);
  float* sl = ds + kT * (kT + 4);  // [64] -lse of the tile's or the walked query rows
  float* sd = sl + kT;             // [64] -delta
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int b = g / p.H, h = g % p.H;
  const float* qg = p.q + b * p.q_sb + h * p.q_sh;
  const float* kg = p.k + b * p.k_sb + h * p.k_sh;
  const float* vg = p.v + b * p.v_sb + h * p.v_sh;
  const float* dg = p.dout + b * p.do_sb + h * p.do_sh;
  const int own0 = tile * kT;
  const float* lse_g = p.w.stat_lse + static_cast<int64_t>(g) * p.w.Sp;
  const float* delta_g = p.w.stat_delta + static_cast<int64_t>(g) * p.w.Sp;
  load_tiles<D>(a1, kKeys ? kg : qg, kKeys ? p.k_ss : p.q_ss, a2, kKeys ? vg : dg, kKeys ? p.v_ss : p.do_ss, own0,
                kKeys ? p.Sk : p.Sq, p.vec);
  if (!kKeys && tid < kT) {
    sl[tid] = lse_g[own0 + tid];
    sd[tid] = delta_g[own0 + tid];
  }
  float acc1[4][4 * DC], acc2[kKeys ? 4 : 1][4 * DC];  // dk or dq; dv
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < 4 * DC; ++c) {
      acc1[i][c] = 0.f;
      if (kKeys) acc2[i][c] = 0.f;
    }
  const int own_block = kKeys ? p.bn : p.bm, walk_block = kKeys ? p.bm : p.bn;
  const int line = own0 / own_block;
  const int lines = kKeys ? p.w.lines_k : p.w.lines_q, cap = kKeys ? p.w.cap_k : p.w.cap_q;
  const int64_t at = static_cast<int64_t>(g) * lines + line;
  const uint16_t* list = (kKeys ? p.w.list_k : p.w.list_q) + at * cap;
  const int walk_len = kKeys ? p.Sq : p.Sk, subs = walk_block / kT;
  const int steps = (kKeys ? p.w.count_k : p.w.count_q)[at] * subs;  // sub-tiles of 64 walked rows
  for (int st = chunk; st < steps; st += p.chunks) {
    const int w0 = (list[st / subs] & 0x3fff) * walk_block + st % subs * kT;
    if (w0 >= walk_len) continue;  // past the end of the last block
    __syncthreads();  // the previous step is consumed
    load_tiles<D>(b1, kKeys ? qg : kg, kKeys ? p.q_ss : p.k_ss, b2, kKeys ? dg : vg, kKeys ? p.do_ss : p.v_ss, w0,
                  walk_len, p.vec);
    if (kKeys && tid < kT) {
      sl[tid] = lse_g[w0 + tid];
      sd[tid] = delta_g[w0 + tid];
    }
    __syncthreads();
    float s[4][4], dp[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[a][c] = dp[a][c] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 x[4], y[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = *reinterpret_cast<const float4*>(&b1[(ty + 16 * c) * LD + d]);
        y[c] = *reinterpret_cast<const float4*>(&a1[(tx + 16 * c) * LD + d]);
      }
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[a][c] = dot4(x[a], y[c], s[a][c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = *reinterpret_cast<const float4*>(&b2[(ty + 16 * c) * LD + d]);
        y[c] = *reinterpret_cast<const float4*>(&a2[(tx + 16 * c) * LD + d]);
      }
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) dp[a][c] = dot4(x[a], y[c], dp[a][c]);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int wr = ty + 16 * a, orow = tx + 16 * c;
        const int qi = kKeys ? wr : orow, key = kKeys ? own0 + orow : w0 + wr;
        // keys past the end (zeros in shared memory) give nothing
        const bool in = key < p.Sk && sl[qi] != -INFINITY;
        const float pr = in ? expf(fmaf(s[a][c], p.scale, sl[qi])) : 0.f;
        if (kKeys) ps[wr * (kT + 4) + orow] = pr;
        ds[wr * (kT + 4) + orow] = in ? pr * (dp[a][c] + sd[qi]) : 0.f;
      }
    __syncthreads();
#pragma unroll 4
    for (int w = 0; w < kT; ++w) {
      const float4 m = *reinterpret_cast<const float4*>(&ds[w * (kT + 4) + ty * 4]);
      const float mv[4] = {m.x, m.y, m.z, m.w};
      float pv[4];
      if (kKeys) {
        const float4 pm = *reinterpret_cast<const float4*>(&ps[w * (kT + 4) + ty * 4]);
        pv[0] = pm.x, pv[1] = pm.y, pv[2] = pm.z, pv[3] = pm.w;
      }
#pragma unroll
      for (int dc = 0; dc < DC; ++dc) {
        const float4 x = *reinterpret_cast<const float4*>(&b1[w * LD + dc * 64 + tx * 4]);
        const float xv[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc1[i][dc * 4 + c] = fmaf(mv[i], xv[c], acc1[i][dc * 4 + c]);
        if (kKeys) {
          const float4 y = *reinterpret_cast<const float4*>(&b2[w * LD + dc * 64 + tx * 4]);
          const float yv[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc2[i][dc * 4 + c] = fmaf(pv[i], yv[c], acc2[i][dc * 4 + c]);
        }
      }
    }
  }
  if (p.chunks > 1) {
    constexpr int kPart = kT * D;
    float* part = p.part + ((static_cast<int64_t>(g) * p.part_tiles + (kKeys ? 2 * tile : 2 * p.tiles_k + tile)) * p.chunks) *
                               kPart;
    // [chunk][dk or dq], then for keys [chunk][dv]; each thread's values side by side
    float4* mine1 = reinterpret_cast<float4*>(part + chunk * kPart) + tid * (4 * DC);
    float4* mine2 = mine1 + static_cast<int64_t>(p.chunks) * kPart / 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        mine1[i * DC + c] = make_float4(acc1[i][4 * c], acc1[i][4 * c + 1], acc1[i][4 * c + 2], acc1[i][4 * c + 3]);
        if (kKeys)
          mine2[i * DC + c] = make_float4(acc2[i][4 * c], acc2[i][4 * c + 1], acc2[i][4 * c + 2], acc2[i][4 * c + 3]);
      }
    __threadfence();
    __syncthreads();
    __shared__ int last;
    if (tid == 0)
      last = atomicAdd(p.part_count + static_cast<int64_t>(g) * gridDim.x + blockIdx.x, 1) == p.chunks - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4 * DC; ++c) {
        acc1[i][c] = 0.f;
        if (kKeys) acc2[i][c] = 0.f;
      }
    for (int ch = 0; ch < p.chunks; ++ch) {  // a chunk's values are in flight together
      const float4* at1 = reinterpret_cast<const float4*>(part + ch * kPart) + tid * (4 * DC);
      const float4* at2 = at1 + static_cast<int64_t>(p.chunks) * kPart / 4;
      float4 x[4 * DC], y[kKeys ? 4 * DC : 1];
#pragma unroll
      for (int j = 0; j < 4 * DC; ++j) {
        x[j] = __ldcg(at1 + j);
        if (kKeys) y[j] = __ldcg(at2 + j);
      }
#pragma unroll
      for (int j = 0; j < 4 * DC; ++j) {
        float* a = &acc1[j / DC][j % DC * 4];
        a[0] += x[j].x, a[1] += x[j].y, a[2] += x[j].z, a[3] += x[j].w;
        if (kKeys) {
          float* v = &acc2[j / DC][j % DC * 4];
          v[0] += y[j].x, v[1] += y[j].y, v[2] += y[j].z, v[3] += y[j].w;
        }
      }
    }
  }
  float* o1 = kKeys ? p.dk + b * p.dk_sb + h * p.dk_sh : p.dq + b * p.dq_sb + h * p.dq_sh;
  float* o2 = p.dv + b * p.dv_sb + h * p.dv_sh;
  const int64_t o1_ss = kKeys ? p.dk_ss : p.dq_ss;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = own0 + ty * 4 + i;
    if (row >= (kKeys ? p.Sk : p.Sq)) continue;
#pragma unroll
    for (int c = 0; c < 4 * DC; ++c) {
      const int d = c / 4 * 64 + tx * 4 + c % 4;
      o1[row * o1_ss + d] = acc1[i][c] * p.scale;
      if (kKeys) o2[row * p.dv_ss + d] = acc2[i][c];
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kSimtThreads, D == 64 ? 2 : 1) bsa_bwd_simt_kernel(const SimtBwdParams p) {
  if (static_cast<int>(blockIdx.x) < p.tiles_k)
    simt_tile<D, true>(p, blockIdx.y, blockIdx.x, blockIdx.z);
  else
    simt_tile<D, false>(p, blockIdx.y, blockIdx.x - p.tiles_k, blockIdx.z);
}

template <int D>
int32_t launch_simt(const SimtBwdParams& p, int tiles_q, int BH, cudaStream_t st) {
  if (const int32_t rc = allow_smem<bsa_bwd_simt_kernel<D>>(kSimtSmem<D>); rc != SAF_OK) return rc;
  const dim3 grid(static_cast<unsigned>(p.tiles_k + tiles_q), static_cast<unsigned>(BH),
                  static_cast<unsigned>(p.chunks));
  bsa_bwd_simt_kernel<D><<<grid, kSimtThreads, kSimtSmem<D>, st>>>(p);
  SAF_CUDA_TRY(cudaGetLastError());
  return SAF_OK;
}

template <typename T>
int32_t launch_prep(const PrepParams& p, int BH, cudaStream_t st) {
  const int words = ((p.nbq > p.nbk ? p.nbq : p.nbk) + 31) / 32;
  const int rows = p.nbq > kGroup ? p.nbq : kGroup;
  const int smem = (kGroup * words + rows + 1) * 4;
  if (smem > 48 * 1024)
    if (const int32_t rc = allow_smem<bwd_prep_kernel<T>>(smem); rc != SAF_OK) return rc;
  const int64_t chunks = p.w.Sp / kRowChunk + (std::is_same<T, __half>::value ? (p.Sk + kRowChunk - 1) / kRowChunk : 0);
  const dim3 grid(static_cast<unsigned>(BH), static_cast<unsigned>(p.groups_k + p.groups_q + chunks));
  bwd_prep_kernel<T><<<grid, 256, smem, st>>>(p);
  SAF_CUDA_TRY(cudaGetLastError());
  return SAF_OK;
}

// Sizes every tensor of a gradient call has to agree on; no device access.
int32_t check_sizes(const saf_tensor4* q, const saf_tensor4* k, int32_t bm, int32_t bn) {
  int32_t rc;
  if ((rc = check_tensor4(q)) != SAF_OK || (rc = check_tensor4(k)) != SAF_OK) return rc;
  if (k->dtype != q->dtype) return SAF_ERR_DTYPE;
  if (k->B != q->B || k->H != q->H || k->D != q->D) return SAF_ERR_SHAPE;
  if (bm <= 0 || bn <= 0) return SAF_ERR_ARG;
  if (q->S > 0x7fffffff || k->S > 0x7fffffff || q->B * q->H > 65535) return SAF_ERR_SHAPE;
  if (q->dtype == SAF_F32) {
    if (bm % kT != 0 || bn % kT != 0 || (q->D != 64 && q->D != 128)) return SAF_ERR_UNSUPPORTED;
  } else if ((bm != 64 && bm != 128) || (bn != 64 && bn != 128) || q->D != 64) {
    return SAF_ERR_UNSUPPORTED;
  }
  if ((q->S + bm - 1) / bm > kMaxBlocks || (k->S + bn - 1) / bn > kMaxBlocks) return SAF_ERR_UNSUPPORTED;
  return SAF_OK;
}

}  // namespace
}  // namespace saf

using namespace saf;

extern "C" size_t saf_bsa_bwd_workspace_bytes(const saf_tensor4* q, const saf_tensor4* k, int32_t block_m,
                                              int32_t block_n) {
  if (check_sizes(q, k, block_m, block_n) != SAF_OK) return 0;
  return layout(q, k, block_m, block_n, nullptr).bytes;
}

extern "C" int32_t saf_bsa_bwd(const saf_tensor4* dout, const saf_tensor4* q, const saf_tensor4* k,
                               const saf_tensor4* v, const saf_tensor4* out, const float* lse,
                               int64_t lse_stride_bh, const saf_tensor4* dq, const saf_tensor4* dk, const saf_tensor4* dv, const int32_t* row_ptr,
                               const int32_t* col_idx, int64_t col_capacity, int32_t block_m, int32_t block_n,
                               float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t rc;
  if ((rc = check_sizes(q, k, block_m, block_n)) != SAF_OK) return rc;
  const saf_tensor4* all[8] = {dout, q, out, dq, k, v, dk, dv};  // the first four by query, the others by key
  for (int i = 0; i < 8; ++i) {
    const saf_tensor4* t = all[i];
    const saf_tensor4* ref = i < 4 ? q : k;
    if ((rc = check_tensor4(t)) != SAF_OK) return rc;
    if (t->dtype != q->dtype) return SAF_ERR_DTYPE;
    if (t->B != ref->B || t->H != ref->H || t->S != ref->S || t->D != ref->D) return SAF_ERR_SHAPE;
    if (q->dtype != SAF_F32 &&
        ((reinterpret_cast<uintptr_t>(t->data) & 15) != 0 || t->stride_s % 8 != 0 ||
         (t->H > 1 && t->stride_h % 8 != 0) || (t->B > 1 && t->stride_b % 8 != 0)))
      return SAF_ERR_STRIDE;
  }
  if (lse == nullptr || row_ptr == nullptr || col_idx == nullptr || col_capacity < 0) return SAF_ERR_ARG;
  if (!(sm_scale > 0.f) || sm_scale > 3.0e38f) return SAF_ERR_ARG;
  if (lse_stride_bh < q->S) return SAF_ERR_STRIDE;
  if (workspace == nullptr || workspace_bytes < saf_bsa_bwd_workspace_bytes(q, k, block_m, block_n))
    return SAF_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return SAF_ERR_STRIDE;
  DeviceScope dev_scope;
  if ((rc = dev_scope.bind(q->data)) != SAF_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int BH = static_cast<int>(q->B * q->H);
  PrepParams pp{};
  pp.out = out->data, pp.dout = dout->data;
  pp.o_sb = out->stride_b, pp.o_sh = out->stride_h, pp.o_ss = out->stride_s;
  pp.d_sb = dout->stride_b, pp.d_sh = dout->stride_h, pp.d_ss = dout->stride_s;
  pp.v = v->data, pp.v_sb = v->stride_b, pp.v_sh = v->stride_h, pp.v_ss = v->stride_s;
  pp.H = static_cast<int>(q->H), pp.D = static_cast<int>(q->D);
  pp.Sq = static_cast<int>(q->S), pp.Sk = static_cast<int>(k->S);
  pp.lse = lse;
  pp.lse_stride = lse_stride_bh;
  pp.lse_factor = 1.f;
  pp.nbq = static_cast<int>((q->S + block_m - 1) / block_m);
  pp.nbk = static_cast<int>((k->S + block_n - 1) / block_n);
  pp.bm = block_m, pp.bn = block_n;
  pp.merge_q = merge_of(q->dtype, block_m), pp.merge_k = merge_of(q->dtype, block_n);
  pp.groups_q = (pp.nbq + kGroup - 1) / kGroup, pp.groups_k = (pp.nbk + kGroup - 1) / kGroup;
  pp.row_ptr = row_ptr, pp.col_idx = col_idx, pp.col_capacity = col_capacity;
  pp.w = layout(q, k, block_m, block_n, static_cast<uint8_t*>(workspace));
  pp.status = device_status_ptr();
  if (pp.status == nullptr) return SAF_ERR_CUDA;
  if (q->dtype != SAF_F32) {
    pp.lse_factor = kLog2e;
    pp.lse_shift = q->dtype == SAF_F16 ? bwd_f16_p_log2_scale() : 0.f;
    pp.items = 1;
    const size_t counters = kCounters + (q->dtype == SAF_F16 ? BH : 0);  // the value maxima follow them
    SAF_CUDA_TRY(cudaMemsetAsync(pp.w.class_count, 0, counters * sizeof(int32_t), st));
    rc = q->dtype == SAF_BF16 ? launch_prep<__nv_bfloat16>(pp, BH, st) : launch_prep<__half>(pp, BH, st);
    if (rc != SAF_OK) return rc;
    return bsa_bwd_sm100(dout, q, k, v, dq, dk, dv, block_m, block_n, sm_scale, pp.w, st);
  }
  if ((rc = launch_prep<float>(pp, BH, st)) != SAF_OK) return rc;
  SimtBwdParams sp{};
  sp.q = static_cast<const float*>(q->data), sp.k = static_cast<const float*>(k->data);
  sp.v = static_cast<const float*>(v->data), sp.dout = static_cast<const float*>(dout->data);
  sp.dq = static_cast<float*>(dq->data), sp.dk = static_cast<float*>(dk->data), sp.dv = static_cast<float*>(dv->data);
  sp.q_sb = q->stride_b, sp.q_sh = q->stride_h, sp.q_ss = q->stride_s;
  sp.k_sb = k->stride_b, sp.k_sh = k->stride_h, sp.k_ss = k->stride_s;
  sp.v_sb = v->stride_b, sp.v_sh = v->stride_h, sp.v_ss = v->stride_s;
  sp.do_sb = dout->stride_b, sp.do_sh = dout->stride_h, sp.do_ss = dout->stride_s;
  sp.dq_sb = dq->stride_b, sp.dq_sh = dq->stride_h, sp.dq_ss = dq->stride_s;
  sp.dk_sb = dk->stride_b, sp.dk_sh = dk->stride_h, sp.dk_ss = dk->stride_s;
  sp.dv_sb = dv->stride_b, sp.dv_sh = dv->stride_h, sp.dv_ss = dv->stride_s;
  sp.H = pp.H, sp.Sq = pp.Sq, sp.Sk = static_cast<int>(k->S);
  sp.bm = block_m, sp.bn = block_n;
  sp.tiles_k = static_cast<int>((k->S + kT - 1) / kT);
  const int tiles_q = static_cast<int>((q->S + kT - 1) / kT);
  sp.scale = sm_scale;
  sp.vec = true;
  for (const saf_tensor4* t : {q, k, v, dout})
    sp.vec = sp.vec && (reinterpret_cast<uintptr_t>(t->data) & 15) == 0 && t->stride_s % 4 == 0 &&
             (t->H == 1 || t->stride_h % 4 == 0) && (t->B == 1 || t->stride_b % 4 == 0);
  sp.w = pp.w;
  sp.chunks = pp.w.chunks, sp.part = pp.w.part, sp.part_count = pp.w.part_count;
  sp.part_tiles = 2 * sp.tiles_k + tiles_q;
  if (sp.chunks > 1)
    SAF_CUDA_TRY(cudaMemsetAsync(sp.part_count, 0, static_cast<size_t>(BH) * (sp.tiles_k + tiles_q) * sizeof(int), st));
  return q->D == 64 ? launch_simt<64>(sp, tiles_q, BH, st) : launch_simt<128>(sp, tiles_q, BH, st);
}
