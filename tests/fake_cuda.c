/* Stand-ins for the CUDA and libmoe_cuda calls of host/moe_host.c, compiled with
 * it into a library that runs on the CPU (test_host_kv_cpu.py): device memory is
 * host memory, copies happen at once, kernels do nothing. What the driver asks
 * for is counted, and an allocation can be made to fail. */
#include <cuda_runtime.h>
#include <stdlib.h>
#include <string.h>

#include "../include/moe_cuda.h"

int fake_fail_in = -1;          /* the n-th cudaMalloc from now fails (0: the next); -1: none */
long fake_largest_ok = -1;      /* bytes that one cudaMalloc may have; -1: any */
int fake_mallocs, fake_live;    /* cudaMalloc calls, and allocations alive */
int fake_unordered;             /* operations on the legacy stream since the host last waited for it */
long fake_ws_per_kv = 0;        /* bytes of attention workspace per position of max_kv */
int fake_short_ws;              /* attention calls that got less workspace than they need */
int fake_cache_dtype = -1;      /* of the last attention call */
long fake_host_limit = -1;      /* bytes that one malloc of the driver may have; -1: any */

static const char* msg = "";

void* fake_malloc(size_t n) { return fake_host_limit >= 0 && n > (size_t)fake_host_limit ? NULL : malloc(n); }

cudaError_t cudaMalloc(void** p, size_t n) {
  ++fake_mallocs;
  const int refuse = fake_fail_in == 0 || (fake_largest_ok >= 0 && n > (size_t)fake_largest_ok);
  if (fake_fail_in >= 0) --fake_fail_in;
  if (refuse) { *p = NULL; return cudaErrorMemoryAllocation; }
  *p = calloc(n ? n : 1, 1);
  ++fake_live;
  return *p ? cudaSuccess : cudaErrorMemoryAllocation;
}
cudaError_t cudaFree(void* p) { if (p) { --fake_live; free(p); } fake_unordered = 0; return cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned f) { (void)f; *p = calloc(n ? n : 1, 1); return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, enum cudaMemcpyKind k) {
  memcpy(d, s, n);
  if (k == cudaMemcpyHostToDevice) ++fake_unordered;      /* pageable: may return before its last piece arrives */
  return cudaSuccess;
}
cudaError_t cudaMemset(void* d, int v, size_t n) { memset(d, v, n); ++fake_unordered; return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, enum cudaMemcpyKind k, cudaStream_t st) {
  (void)k;
  memcpy(d, s, n);
  if (!st) ++fake_unordered;
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t st) {
  memset(d, v, n);
  if (!st) ++fake_unordered;
  return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize(void) { fake_unordered = 0; return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t st) { if (!st) fake_unordered = 0; return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned f) { (void)f; *s = (cudaStream_t)malloc(8); return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t s) { free(s); return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { (void)d; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t e) { return e == cudaErrorMemoryAllocation ? "out of memory" : "error"; }

const char* moe_cuda_last_error(void) { return msg; }
int moe_kv_plan_dev(const int* past, const int* fresh, int n, int ps, int np, const int* f, int nf, const int* h, int* t, int mp,
                    int* kv, int* a, int* b, int* c, int cap, int* ho, int* st, void* s) {
  return MOE_OK;
}
int moe_qk_norm_rope_dev(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, int dt, int rows,
                         int nq, const float* qn, const float* kn, float eps, const float* r, int rot, int len, const int* pos,
                         const int* slot, void* o, long long ldo, const MoeKvCache* c, void* s) {
  return MOE_OK;
}
size_t moe_paged_attention_workspace(int rows, int nq, const MoeKvCache* c, int max_kv) { return (size_t)(fake_ws_per_kv * max_kv); }
int moe_paged_attention_dev(const void* q, long long ldq, const MoeKvCache* c, const int* t, int n, int mp, const int* seq,
                            const int* pos, int rows, int nq, int max_kv, float scale, void* o, long long ldo, float* lse, void* ws,
                            size_t bytes, void* s) {
  const size_t need = moe_paged_attention_workspace(rows, nq, c, max_kv);
  if (need && (!ws || bytes < need)) ++fake_short_ws;
  fake_cache_dtype = c->dtype;
  return MOE_OK;
}
int moe_synth_normal_dev(uint64_t seed, uint64_t off, size_t n, float std, float* out, void* s) { return MOE_OK; }
