// rope.cu -- rotary positions on q and k in one launch (saf_rope).
//
// The first text_len tokens are copied; token text_len + t has its first R
// channels rotated pair by pair through the angles of table row t:
//   a' = a cos - b sin,  b' = b cos + a sin
// with pairs (2m, 2m + 1) (interleaved) or (m, m + R/2) (half); channels R..D
// are copied.  The gradient of the rotation is its transpose, the same with
// -sin.  Products and sums in fp32, one rounding to the stored type.
//
// Bound by HBM: q and k are read and written once, in 16-byte pieces.  A
// thread owns one piece (two in the half layout) of one token's row and walks
// up to kPlanes heads of q or of k with it: cos and sin are loaded once for
// them, the heads' loads are all in flight before the first store (so a tensor
// may be rotated in place), and a head costs one pointer addition.
// Measured with 1, 2, 4, 8 heads a thread: 60 heads of 17776 tokens, D = 64,
// bf16, interleaved 118, 84.1, 84.6, 86.3 us (4: 6.5 TB/s, the copy's rate);
// a long strided half layout in f16 174, 133, 119, 133 us.
#include "saf_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace saf {
namespace {

constexpr int kPlanes = 4;

struct RopeParams {
  const void* q;
  const void* k;
  void* oq;
  void* ok;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, oq_sb, oq_sh, oq_ss, ok_sb, ok_sh, ok_ss;
  int Hq, Hk, groups_q, groups;  // thread groups over the heads of q, of q and k
  int64_t S, text;
  int D, R, units;  // units: pieces of a row, one per thread
  const float* cs;
  const float* sn;
  int64_t table_sb;
  float sign;
};

__device__ __forceinline__ float2 unpack(uint32_t x, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t x, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, const __nv_bfloat16*) { return pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint32_t pack(float lo, float hi, const __half*) { return pack_f16x2(lo, hi); }

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = a * c - b * s;
  b = b * c + a * s;
  a = x;
}

// A 16-byte piece holding whole pairs (interleaved).
template <typename T>
__device__ __forceinline__ void turn_piece(uint32_t (&x)[4], const float* cs, const float* sn) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 2) {
      float2 v = unpack(x[w], static_cast<const T*>(nullptr));
      turn(v.x, v.y, cs[w], sn[w]);
      x[w] = pack(v.x, v.y, static_cast<const T*>(nullptr));
    } else if (w % 2 == 0) {
      float a = __uint_as_float(x[w]), b = __uint_as_float(x[w + 1]);
      turn(a, b, cs[w / 2], sn[w / 2]);
      x[w] = __float_as_uint(a);
      x[w + 1] = __float_as_uint(b);
    }
  }
}
// Two 16-byte pieces, first and second channels of their pairs (half layout).
template <typename T>
__device__ __forceinline__ void turn_pieces(uint32_t (&x)[4], uint32_t (&y)[4], const float* cs, const float* sn) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 2) {
      float2 a = unpack(x[w], static_cast<const T*>(nullptr)), b = unpack(y[w], static_cast<const T*>(nullptr));
      turn(a.x, b.x, cs[2 * w], sn[2 * w]);
      turn(a.y, b.y, cs[2 * w + 1], sn[2 * w + 1]);
      x[w] = pack(a.x, a.y, static_cast<const T*>(nullptr));
      y[w] = pack(b.x, b.y, static_cast<const T*>(nullptr));
    } else {
      float a = __uint_as_float(x[w]), b = __uint_as_float(y[w]);
      turn(a, b, cs[w], sn[w]);
      x[w] = __float_as_uint(a);
      y[w] = __float_as_uint(b);
    }
  }
}

__device__ __forceinline__ void load_piece(uint32_t (&x)[4], const void* src) {
  const uint4 v = *static_cast<const uint4*>(src);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void store_piece(void* dst, const uint32_t (&x)[4]) {
  *static_cast<uint4*>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
}

// This thread's heads: base pointers at its token, head stride, count.
template <typename T>
struct Heads {
  const T* src;
  T* dst;
  int64_t src_sh, dst_sh;
  int n;
};
template <typename T>
__device__ __forceinline__ Heads<T> heads_of(const RopeParams& p, int b, int group, int64_t s) {
  Heads<T> h;
  if (group < p.groups_q) {
    const int h0 = group * kPlanes;
    h.src = static_cast<const T*>(p.q) + b * p.q_sb + h0 * p.q_sh + s * p.q_ss;
    h.dst = static_cast<T*>(p.oq) + b * p.oq_sb + h0 * p.oq_sh + s * p.oq_ss;
    h.src_sh = p.q_sh, h.dst_sh = p.oq_sh, h.n = min(kPlanes, p.Hq - h0);
  } else {
    const int h0 = (group - p.groups_q) * kPlanes;
    h.src = static_cast<const T*>(p.k) + b * p.k_sb + h0 * p.k_sh + s * p.k_ss;
    h.dst = static_cast<T*>(p.ok) + b * p.ok_sb + h0 * p.ok_sh + s * p.ok_ss;
    h.src_sh = p.k_sh, h.dst_sh = p.ok_sh, h.n = min(kPlanes, p.Hk - h0);
  }
  return h;
}

// One thread per (token, unit); blockIdx.y = batch x head group.  A unit is a
// 16-byte piece of V channels (interleaved, or copied), or below R the two
// pieces R/2 apart that make V pairs (half layout).
template <typename T, bool kHalf, int V>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
  static_assert(V * sizeof(T) == 16, "16-byte pieces");
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t s = idx / p.units;
  if (s >= p.S) return;
  const int u = static_cast<int>(idx - s * p.units);
  const int b = blockIdx.y / p.groups, group = blockIdx.y - b * p.groups;
  const int turned = kHalf ? p.R / (2 * V) : p.R / V;
  const bool rotate = u < turned && s >= p.text;
  const bool two = kHalf && u < turned;
  const int c0 = kHalf && !two ? p.R + (u - turned) * V : u * V;
  constexpr int NA = kHalf ? V : V / 2;  // angles of a unit
  float cs[NA], sn[NA];
  if (rotate) {
    const int64_t at = b * p.table_sb + (s - p.text) * (p.R / 2) + (kHalf ? c0 : c0 / 2);
#pragma unroll
    for (int i = 0; i < NA; i += 2) {
      const float2 c = __ldg(reinterpret_cast<const float2*>(p.cs + at + i));
      const float2 w = __ldg(reinterpret_cast<const float2*>(p.sn + at + i));
      cs[i] = c.x, cs[i + 1] = c.y;
      sn[i] = w.x * p.sign, sn[i + 1] = w.y * p.sign;
    }
  }
  const Heads<T> h = heads_of<T>(p, b, group, s);
  uint32_t x[kPlanes][4], y[kHalf ? kPlanes : 1][4];
  const T* src = h.src + c0;
#pragma unroll
  for (int i = 0; i < kPlanes; ++i) {
    if (i < h.n) {
      load_piece(x[i], src);
      if constexpr (kHalf)
        if (two) load_piece(y[i], src + p.R / 2);
    }
    src += h.src_sh;
  }
  T* dst = h.dst + c0;
#pragma unroll
  for (int i = 0; i < kPlanes; ++i) {
    if (i < h.n) {
      if (rotate) {
        if constexpr (kHalf)
          turn_pieces<T>(x[i], y[i], cs, sn);
        else
          turn_piece<T>(x[i], cs, sn);
      }
      store_piece(dst, x[i]);
      if constexpr (kHalf)
        if (two) store_piece(dst + p.R / 2, y[i]);
    }
    dst += h.dst_sh;
  }
}

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return static_cast<float>(x);
}
__device__ __forceinline__ void put(float* d, float x) { *d = x; }
__device__ __forceinline__ void put(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half* d, float x) { *d = __float2half_rn(x); }

// Rows without whole, aligned 16-byte pieces: one pair (or copied channel) a
// thread, single elements.
template <typename T, bool kHalf>
__global__ void __launch_bounds__(256) rope_element_kernel(const RopeParams p) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t s = idx / p.units;
  if (s >= p.S) return;
  const int u = static_cast<int>(idx - s * p.units);
  const int b = blockIdx.y / p.groups, group = blockIdx.y - b * p.groups;
  const bool pair = u < p.R / 2;
  const int c0 = !pair ? u + p.R / 2 : kHalf ? u : 2 * u;
  const int c1 = kHalf ? c0 + p.R / 2 : c0 + 1;
  float cs = 1.f, sn = 0.f;
  const bool rotate = pair && s >= p.text;
  if (rotate) {
    const int64_t at = b * p.table_sb + (s - p.text) * (p.R / 2) + u;
    cs = __ldg(p.cs + at);
    sn = __ldg(p.sn + at) * p.sign;
  }
  const Heads<T> h = heads_of<T>(p, b, group, s);
  for (int i = 0; i < h.n; ++i) {
    const T* src = h.src + i * h.src_sh;
    T* dst = h.dst + i * h.dst_sh;
    const T x0 = src[c0];
    if (!pair) {
      dst[c0] = x0;
      continue;
    }
    const T x1 = src[c1];
    if (rotate) {
      float a = to_f(x0), c = to_f(x1);
      turn(a, c, cs, sn);
      put(dst + c0, a);
      put(dst + c1, c);
    } else {
      dst[c0] = x0;
      dst[c1] = x1;
    }
  }
}

template <typename T, bool kHalf>
int32_t launch(RopeParams& p, int64_t B, bool pieces, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  p.units = pieces ? (kHalf ? p.R / (2 * V) : p.R / V) + (p.D - p.R) / V : p.R / 2 + (p.D - p.R);
  const int64_t bx = (p.S * p.units + 255) / 256, by = B * p.groups;
  if (bx > 0x7fffffff || by > 65535) return SAF_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  if (pieces)
    rope_kernel<T, kHalf, V><<<grid, 256, 0, stream>>>(p);
  else
    rope_element_kernel<T, kHalf><<<grid, 256, 0, stream>>>(p);
  SAF_CUDA_TRY(cudaGetLastError());
  return SAF_OK;
}

// 16-byte pieces need R (its halves in the half layout) and D - R to be whole
// numbers of them, and every row and table row aligned.
template <typename T>
int32_t dispatch(RopeParams& p, int64_t B, bool half, bool aligned, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool pieces = aligned && p.D % V == 0 && p.R % (half ? 2 * V : V) == 0;
  return half ? launch<T, true>(p, B, pieces, stream) : launch<T, false>(p, B, pieces, stream);
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
  if (q->H > 65535 || (k != nullptr && k->H > 65535)) return SAF_ERR_SHAPE;
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
  p.Hk = k != nullptr ? static_cast<int>(k->H) : 0;
  p.groups_q = (p.Hq + kPlanes - 1) / kPlanes;
  p.groups = p.groups_q + (p.Hk + kPlanes - 1) / kPlanes;
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
                       ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 7) == 0 &&
                       rotary_dim / 2 % 2 == 0 && (q->B == 1 || table_stride_b % 2 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = half_layout != 0;
  if (q->dtype == SAF_BF16) return dispatch<__nv_bfloat16>(p, q->B, half, aligned, st);
  if (q->dtype == SAF_F16) return dispatch<__half>(p, q->B, half, aligned, st);
  return dispatch<float>(p, q->B, half, aligned, st);
}
