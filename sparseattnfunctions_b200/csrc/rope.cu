// rope.cu -- rotary positions on q and k in one launch (saf_rope).
//
// The first text_len tokens are copied; token text_len + t has its first R
// channels rotated pair by pair through the angles of table row t:
//   a' = a cos - b sin,  b' = b cos + a sin
// with pairs (2m, 2m + 1) (interleaved) or (m, m + R/2) (half); channels R..D
// are copied.  The gradient of the rotation is its transpose, the same with
// -sin.  Products and sums in fp32, one rounding to the stored type.
//
// Bound by HBM: q and k are read and written once (16-byte accesses); a
// token's cos and sin are loaded once by the thread that owns that piece of
// the row and reused over up to kPlanes heads of q and k, whose loads are all
// in flight before the first store (so a tensor may be rotated in place).
#include "saf_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace saf {
namespace {

constexpr int kPlanes = 8;  // heads (of q, then of k) one thread handles

struct RopeParams {
  const void* q;
  const void* k;
  void* oq;
  void* ok;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, oq_sb, oq_sh, oq_ss, ok_sb, ok_sh, ok_ss;
  int Hq, planes, groups;  // heads of q, of q and k together, thread groups over them
  int64_t S, text;
  int D, R, units;  // units: pieces of a row, one per thread
  const float* cs;
  const float* sn;
  int64_t table_sb;
  float sign;
};

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return static_cast<float>(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
  return __float2half_rn(x);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// One thread per (token, unit); blockIdx.y = batch x plane group.  A unit is V
// copied channels, or below R either V channels that hold whole pairs
// (interleaved, 16-byte pieces) or the two pieces of V channels that make V
// pairs (R/2 apart in the half layout, neighbours in the interleaved one with
// V = 1).  V is 16 bytes when every piece is whole and aligned, else 1.
template <typename T, bool kHalf, int V>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t s = idx / p.units;
  if (s >= p.S) return;
  const int u = static_cast<int>(idx % p.units);
  const int b = blockIdx.y / p.groups, plane0 = (blockIdx.y % p.groups) * kPlanes;
  // the unit's first channel, and its second piece's in the half layout
  constexpr bool kTwo = kHalf || V == 1;  // a pair's channels come from two pieces
  const int turned = kTwo ? p.R / (2 * V) : p.R / V;
  const bool rot_unit = u < turned;
  const int c0 = !rot_unit ? p.R + (u - turned) * V : kHalf || !kTwo ? u * V : 2 * u;
  const int c1 = kHalf ? c0 + p.R / 2 : c0 + 1;
  constexpr int NA = kTwo ? V : V / 2;  // angles of a unit
  const bool two = kTwo && rot_unit;
  const bool rotate = rot_unit && s >= p.text;
  float cs[NA], sn[NA];
  if (rotate) {
    const int64_t at = b * p.table_sb + (s - p.text) * (p.R / 2) + (kHalf ? c0 : c0 / 2);
    if constexpr (NA % 4 == 0) {
#pragma unroll
      for (int i = 0; i < NA; i += 4) {
        const float4 c = __ldg(reinterpret_cast<const float4*>(p.cs + at + i));
        const float4 w = __ldg(reinterpret_cast<const float4*>(p.sn + at + i));
        cs[i] = c.x, cs[i + 1] = c.y, cs[i + 2] = c.z, cs[i + 3] = c.w;
        sn[i] = w.x, sn[i + 1] = w.y, sn[i + 2] = w.z, sn[i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        cs[i] = __ldg(p.cs + at + i);
        sn[i] = __ldg(p.sn + at + i);
      }
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) sn[i] *= p.sign;
  }
  using W = Vec<T, V>;
  W x0[kPlanes], x1[kTwo ? kPlanes : 1];
#pragma unroll
  for (int i = 0; i < kPlanes; ++i) {
    const int pl = plane0 + i;
    if (pl >= p.planes) break;
    const T* src = pl < p.Hq ? static_cast<const T*>(p.q) + b * p.q_sb + pl * p.q_sh + s * p.q_ss
                             : static_cast<const T*>(p.k) + b * p.k_sb + (pl - p.Hq) * p.k_sh + s * p.k_ss;
    x0[i] = *reinterpret_cast<const W*>(src + c0);
    if constexpr (kTwo)
      if (two) x1[i] = *reinterpret_cast<const W*>(src + c1);
  }
#pragma unroll
  for (int i = 0; i < kPlanes; ++i) {
    const int pl = plane0 + i;
    if (pl >= p.planes) break;
    T* dst = pl < p.Hq ? static_cast<T*>(p.oq) + b * p.oq_sb + pl * p.oq_sh + s * p.oq_ss
                       : static_cast<T*>(p.ok) + b * p.ok_sb + (pl - p.Hq) * p.ok_sh + s * p.ok_ss;
    if (rotate) {
#pragma unroll
      for (int m = 0; m < NA; ++m) {
        T& lo = kTwo ? x0[i].v[m] : x0[i].v[2 * m % V];
        T& hi = kTwo ? x1[kTwo ? i : 0].v[m] : x0[i].v[(2 * m + 1) % V];
        const float a = to_f(lo), c = to_f(hi);
        lo = from_f<T>(a * cs[m] - c * sn[m]);
        hi = from_f<T>(c * cs[m] + a * sn[m]);
      }
    }
    *reinterpret_cast<W*>(dst + c0) = x0[i];
    if constexpr (kTwo)
      if (two) *reinterpret_cast<W*>(dst + c1) = x1[i];
  }
}

template <typename T, bool kHalf, int V>
int32_t launch(RopeParams& p, int64_t B, cudaStream_t stream) {
  p.units = (kHalf || V == 1 ? p.R / (2 * V) : p.R / V) + (p.D - p.R) / V;
  const int64_t threads = p.S * p.units;
  const int64_t by = B * p.groups, bx = (threads + 255) / 256;
  if (bx > 0x7fffffff || by > 65535) return SAF_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  rope_kernel<T, kHalf, V><<<grid, 256, 0, stream>>>(p);
  SAF_CUDA_TRY(cudaGetLastError());
  return SAF_OK;
}

// The vector form needs whole 16-byte pieces: R and D - R split into pieces of
// V channels (each half of R in the half layout), every row and the table rows
// 16-byte aligned.  Anything else takes one pair (or copied channel) a thread,
// with single-element accesses.
template <typename T>
int32_t dispatch(RopeParams& p, int64_t B, bool half, bool aligned, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = p.D % V == 0 && p.R % (half ? 2 * V : V) == 0;
  if (half) return aligned && whole ? launch<T, true, V>(p, B, stream) : launch<T, true, 1>(p, B, stream);
  return aligned && whole ? launch<T, false, V>(p, B, stream) : launch<T, false, 1>(p, B, stream);
}

}  // namespace
}  // namespace saf

using namespace saf;

extern "C" int32_t saf_rope(const saf_tensor4* q, const saf_tensor4* k, const saf_tensor4* out_q,
                            const saf_tensor4* out_k, const float* cos_table, const float* sin_table,
                            int64_t table_stride_b, int64_t text_len, int32_t rotary_dim, int32_t half_layout,
                            int32_t inverse, void* stream) {
  int32_t rc;
  if ((rc = check_tensor4(q)) != SAF_OK || (rc = check_tensor4(out_q)) != SAF_OK) return rc;
  if ((k == nullptr) != (out_k == nullptr)) return SAF_ERR_ARG;
  if (k != nullptr && ((rc = check_tensor4(k)) != SAF_OK || (rc = check_tensor4(out_k)) != SAF_OK)) return rc;
  if (out_q->dtype != q->dtype || (k != nullptr && (k->dtype != q->dtype || out_k->dtype != q->dtype)))
    return SAF_ERR_DTYPE;
  auto same = [](const saf_tensor4* a, const saf_tensor4* b) {
    return a->B == b->B && a->H == b->H && a->S == b->S && a->D == b->D;
  };
  if (!same(q, out_q)) return SAF_ERR_SHAPE;
  if (k != nullptr && (!same(k, out_k) || k->B != q->B || k->S != q->S || k->D != q->D)) return SAF_ERR_SHAPE;
  if (text_len < q->S && (cos_table == nullptr || sin_table == nullptr)) return SAF_ERR_ARG;
  if (text_len < 0 || text_len > q->S || table_stride_b < 0) return SAF_ERR_SHAPE;
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > q->D || q->D > 65536) return SAF_ERR_SHAPE;
  const int64_t planes = q->H + (k != nullptr ? k->H : 0);
  if (planes > 65535) return SAF_ERR_SHAPE;
  DeviceScope dev_scope;
  if ((rc = dev_scope.bind(q->data)) != SAF_OK) return rc;
  RopeParams p{};
  p.q = q->data;
  p.oq = out_q->data;
  p.q_sb = q->stride_b, p.q_sh = q->stride_h, p.q_ss = q->stride_s;
  p.oq_sb = out_q->stride_b, p.oq_sh = out_q->stride_h, p.oq_ss = out_q->stride_s;
  if (k != nullptr) {
    p.k = k->data;
    p.ok = out_k->data;
    p.k_sb = k->stride_b, p.k_sh = k->stride_h, p.k_ss = k->stride_s;
    p.ok_sb = out_k->stride_b, p.ok_sh = out_k->stride_h, p.ok_ss = out_k->stride_s;
  }
  p.Hq = static_cast<int>(q->H);
  p.planes = static_cast<int>(planes);
  p.groups = (p.planes + kPlanes - 1) / kPlanes;
  p.S = q->S;
  p.text = text_len;
  p.D = static_cast<int>(q->D);
  p.R = rotary_dim;
  p.cs = cos_table;
  p.sn = sin_table;
  p.table_sb = table_stride_b;
  p.sign = inverse != 0 ? -1.f : 1.f;
  const int eb = elem_bytes(q->dtype);
  auto rows_aligned = [&](const saf_tensor4* t) {
    return t == nullptr || ((reinterpret_cast<uintptr_t>(t->data) & 15) == 0 && t->stride_s * eb % 16 == 0 &&
                            (t->H == 1 || t->stride_h * eb % 16 == 0) && (t->B == 1 || t->stride_b * eb % 16 == 0));
  };
  const bool aligned = rows_aligned(q) && rows_aligned(k) && rows_aligned(out_q) && rows_aligned(out_k) &&
                       ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) == 0 &&
                       rotary_dim / 2 % 4 == 0 && (q->B == 1 || table_stride_b % 4 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = half_layout != 0;
  if (q->dtype == SAF_BF16) return dispatch<__nv_bfloat16>(p, q->B, half, aligned, st);
  if (q->dtype == SAF_F16) return dispatch<__half>(p, q->B, half, aligned, st);
  return dispatch<float>(p, q->B, half, aligned, st);
}
