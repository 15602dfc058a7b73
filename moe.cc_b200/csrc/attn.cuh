// attn.cuh — what the attention-side entry points (kv_plan.cu, qk_rope.cu,
// paged_attn.cu, expert_route.cu) share: element types, argument errors, the
// device of a call's pointers, and small device helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/moe_cuda.h"
#include "common.cuh"

namespace moe {

int set_error_message(int code, const char* msg);   // runtime.cu

namespace at {

inline int fail(int code, const char* fmt, ...) {
  char buf[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error_message(code, buf);
}

inline int elem_size(int dtype) {
  return dtype == MOE_DTYPE_F32 ? 4 : dtype == MOE_DTYPE_F16 || dtype == MOE_DTYPE_BF16 ? 2 : 0;
}

// The call runs on the device that holds `p`, whatever device is current;
// the current device is put back when the call returns. Ordinary host memory
// is refused here, before a kernel would fault on it.
class OnDeviceOf {
 public:
  ~OnDeviceOf() { if (back_ >= 0) cudaSetDevice(back_); }
  int enter(const void* p, const char* who) {
    cudaPointerAttributes a{};
    cudaError_t e = cudaPointerGetAttributes(&a, p);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    if (a.type == cudaMemoryTypeUnregistered)
      return fail(MOE_ERR_INVALID, "%s: the pointers must be device memory", who);
    int cur = 0;
    if ((e = cudaGetDevice(&cur)) != cudaSuccess) return fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    dev_ = cur;
    if (a.type != cudaMemoryTypeHost && a.device != cur) {
      if ((e = cudaSetDevice(a.device)) != cudaSuccess)
        return fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
      back_ = cur;
      dev_ = a.device;
    }
    return MOE_OK;
  }
  int device() const { return dev_; }

 private:
  int back_ = -1, dev_ = 0;
};

inline int launched(cudaError_t e, const char* who) {
  if (e == cudaSuccess) return MOE_OK;
  cudaGetLastError();
  return fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

// The cache description every entry point that touches it checks alike.
// Strides count elements; rows of head_dim elements are contiguous and start
// on 16-byte boundaries, so that they move in 16-byte pieces.
inline int check_cache(const MoeKvCache* c, const char* who) {
  if (!c || !c->k || !c->v) return fail(MOE_ERR_INVALID, "%s: no cache", who);
  const int es = elem_size(c->dtype);
  if (!es) return fail(MOE_ERR_INVALID, "%s: cache dtype %d (f32, f16 or bf16 is wanted)", who, c->dtype);
  if (c->n_pages < 1 || c->page_size < 1 || c->n_kv < 1)
    return fail(MOE_ERR_INVALID, "%s: cache of %d pages x %d tokens x %d heads", who, c->n_pages, c->page_size, c->n_kv);
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
    return fail(MOE_ERR_UNSUPPORTED, "%s: head_dim %d (multiples of 8 from 8 to 256)", who, c->head_dim);
  if ((long long)c->n_pages * c->page_size > INT32_MAX)
    return fail(MOE_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", who);
  const int q = 16 / es;
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || c->page_stride % q || c->token_stride % q || c->head_stride % q)
    return fail(MOE_ERR_INVALID, "%s: cache rows must start on 16-byte boundaries", who);
  if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
    return fail(MOE_ERR_INVALID, "%s: negative cache stride", who);
  return MOE_OK;
}

// whether `rows` rows of two operands, n elements of e bytes each and ld from
// one to the next, may share a byte: their ranges meet, and they are not
// columns of one matrix that lie beside each other
inline bool overlap(const void* p, long long ldp, long long np, int ep, const void* r, long long ldr, long long nr,
                    int er, int rows) {
  const long long p0 = (long long)(uintptr_t)p, r0 = (long long)(uintptr_t)r, sp = ldp * ep, sr = ldr * er;
  const long long bp = np * ep, br = nr * er;
  if (p0 + (rows - 1) * sp + bp <= r0 || r0 + (rows - 1) * sr + br <= p0) return false;
  if (sp != sr || sp <= 0) return true;
  const long long d = ((r0 - p0) % sp + sp) % sp;       // from a row of p to the next row of r
  return d < bp || d + br > sp;
}

// n / d for 0 <= n < 2^31 by one multiply: with l = ceil(log2 d) and
// m = floor(2^(31+l) / d) + 1, the excess e = m d - 2^(31+l) lies in (0, d],
// so e n < 2^(31+l) and floor(n m / 2^(31+l)) = floor(n / d).
struct FastDiv {
  unsigned d, m, s;
  FastDiv() = default;
  explicit FastDiv(unsigned div) : d(div) {
    unsigned l = 0;
    while ((1ull << l) < div) ++l;
    s = 31 + l;
    m = (unsigned)((1ull << s) / div + 1);
  }
  __host__ __device__ unsigned div(unsigned n) const { return (unsigned)(((unsigned long long)n * m) >> s); }
};

// ---- element conversions (one rounding, to nearest even) --------------------
template <typename T> struct Vec4;       // four elements, loaded and stored together
template <> struct Vec4<float> {
  using raw = float4;
  static __device__ __forceinline__ void get(const raw& r, float* f) { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
  static __device__ __forceinline__ raw put(const float* f) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Vec4<__nv_bfloat16> {
  using raw = uint2;
  static __device__ __forceinline__ void get(const raw& r, float* f) {
    f[0] = __uint_as_float(r.x << 16); f[1] = __uint_as_float(r.x & 0xffff0000u);
    f[2] = __uint_as_float(r.y << 16); f[3] = __uint_as_float(r.y & 0xffff0000u);
  }
  static __device__ __forceinline__ raw put(const float* f) {
    __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<unsigned*>(&a), *reinterpret_cast<unsigned*>(&b));
  }
};
template <> struct Vec4<__half> {
  using raw = uint2;
  static __device__ __forceinline__ void get(const raw& r, float* f) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
  static __device__ __forceinline__ raw put(const float* f) {
    __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<unsigned*>(&a), *reinterpret_cast<unsigned*>(&b));
  }
};

}  // namespace at
}  // namespace moe
