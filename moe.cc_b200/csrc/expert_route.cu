// expert_route.cu — moe_route_dev: expert routing from router logits, for the
// routings that the resident layers' own router (softmax over the top k,
// test_model_trace.c:463-490) does not cover. Its lists are what moe_ffn takes
// with MOE_FFN_GIVEN_TOPK.
//
//   s_e = exp(x_e - max x) / sum exp(x - max x)   or   1 / (1 + exp(-x_e))
//   c_e = s_e + bias_e                            the choice goes by c, the weights by s
//   groups: the sum of a group's best one or two c; only the best groups stay
//   top k by c, ties to the lower index; p = s, divided by the sum of the
//   chosen s if wanted, times a factor
//
// Scores, choices and sums are held in 64 bits: the choice is an ordering, and
// in fp32 two different sigmoid scores near 1 (or scores plus a bias) round to
// the same number often enough to change which expert is chosen. An exp in
// double costs little here: E of them per token, at B200's 64 double-precision
// lanes per SM. Without a bias or groups the order of the scores is the order
// of the logits, and then only the chosen experts' scores are computed (and
// the softmax's sum, where the weights are not renormalised).
//
// One warp routes one token: expert j * 32 + lane in lane `lane`. A round of
// the selection takes the largest 64-bit key by two 32-bit warp reductions and
// the lowest index that has it by a third, so k rounds are k times about 40
// instructions. Small calls are bound by the launch and those rounds' latency.
#include "attn.cuh"

namespace moe {
namespace {

constexpr int kWarps = 4;

struct RouteArgs {
  const void* x;
  const float* bias;
  int* idx;
  float* p;
  long long ld;
  int rows, E, softmax, groups, keep, group_top, topk, renorm, lanes_per_group, group_size;
  double factor;
};

// order-preserving 64-bit key of a choice; 0 is below every number's key
__device__ __forceinline__ unsigned long long key_of(double c) {
  const long long b = __double_as_longlong(c + 0.0);      // -0 and 0 are one value
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

template <typename T> __device__ __forceinline__ float logit(const void* x, long long i);
template <> __device__ __forceinline__ float logit<float>(const void* x, long long i) { return ((const float*)x)[i]; }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(const void* x, long long i) { return __bfloat162float(((const __nv_bfloat16*)x)[i]); }
template <> __device__ __forceinline__ float logit<__half>(const void* x, long long i) { return __half2float(((const __half*)x)[i]); }

// exp(x - top) with x = top = +inf counted as 1
__device__ __forceinline__ double weight_of(float x, float top) { return x == top ? 1.0 : exp((double)x - (double)top); }
__device__ __forceinline__ double sigmoid64(float x) { return 1.0 / (1.0 + exp(-(double)x)); }

// EPL experts a lane; SCORED: the choice needs every score (bias or groups)
template <typename T, int EPL, bool SCORED>
__global__ void __launch_bounds__(kWarps * 32) expert_route_kernel(const RouteArgs a) {
  pdl_wait();
  pdl_launch();
  extern __shared__ double choice_sm[];                    // groups: [kWarps][EPL * 32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = (long long)blockIdx.x * kWarps + warp;
  if (t >= a.rows) return;
  float x[EPL];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = j * 32 + lane;
    x[j] = e < a.E ? logit<T>(a.x, t * a.ld + e) : -INFINITY;
    if (!(x[j] > -INFINITY)) x[j] = -INFINITY;            // NaN: never chosen, as -inf
    top = fmaxf(top, x[j]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));

  double total = 1.0;
  unsigned long long key[EPL];
  if constexpr (SCORED) {
    double c[EPL];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const bool in = x[j] > -INFINITY;
      c[j] = !in ? 0.0 : a.softmax ? weight_of(x[j], top) : sigmoid64(x[j]);
      sum += c[j];
    }
    if (a.softmax) total = warp_sum64(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (a.softmax) c[j] = c[j] / total;
      if (a.bias && j * 32 + lane < a.E) c[j] += (double)a.bias[j * 32 + lane];
      const bool in = x[j] > -INFINITY && c[j] > -INFINITY;    // a NaN or -inf bias hides its expert
      if (!in) c[j] = -INFINITY;
      key[j] = in ? key_of(c[j]) : 0ull;
    }
    if (a.groups > 1) {
      double* mine = choice_sm + warp * (EPL * 32);
#pragma unroll
      for (int j = 0; j < EPL; ++j) mine[j * 32 + lane] = c[j];
      __syncwarp();
      // lanes_per_group lanes look through a group and merge their best two
      const int lpg = a.lanes_per_group, grp = lane / lpg;
      double b0 = -INFINITY, b1 = -INFINITY;
      if (grp < a.groups)
        for (int i = lane % lpg; i < a.group_size; i += lpg) {
          const double v = mine[grp * a.group_size + i];
          if (v > b0) { b1 = b0; b0 = v; } else if (v > b1) b1 = v;
        }
      for (int o = 1; o < lpg; o <<= 1) {
        const double o0 = __shfl_xor_sync(~0u, b0, o), o1 = __shfl_xor_sync(~0u, b1, o);
        const double lo = b0 > o0 ? o0 : b0;
        b1 = fmax(lo, fmax(b1, o1));
        b0 = fmax(b0, o0);
      }
      const double gs = b0 + (a.group_top == 2 && b1 > -INFINITY ? b1 : 0.0);
      // a group stays if fewer than `keep` groups come before it
      int before = 0;
      for (int h = 0; h < a.groups; ++h) {
        const double v = __shfl_sync(~0u, gs, h * lpg);
        before += v > gs || (v == gs && h < grp);
      }
      const unsigned stays = __ballot_sync(~0u, grp < a.groups && before < a.keep && lane % lpg == 0);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = j * 32 + lane, ge = e / a.group_size;
        if (e >= a.E || !((stays >> (ge * lpg)) & 1)) key[j] = 0ull;
      }
    }
  } else {
    if (a.softmax && !a.renorm) {
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) sum += x[j] > -INFINITY ? weight_of(x[j], top) : 0.0;
      total = warp_sum64(sum);
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int b = __float_as_int(x[j] + 0.0f);
      const unsigned k = (unsigned)b ^ (b < 0 ? ~0u : 1u << 31);
      key[j] = x[j] > -INFINITY ? k : 0u;
    }
  }

  // k rounds; lane r keeps the r-th choice
  int chosen = -1;
  for (int r = 0; r < a.topk; ++r) {
    unsigned long long best = key[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < EPL; ++j)
      if (key[j] > best) { best = key[j]; at = j; }
    bool cand = true;
    unsigned any;
    if constexpr (SCORED) {
      const unsigned hi = (unsigned)(best >> 32), top_hi = __reduce_max_sync(~0u, hi);
      cand = hi == top_hi;
      any = top_hi;
      const unsigned lo = cand ? (unsigned)best : 0u, top_lo = __reduce_max_sync(~0u, lo);
      cand = cand && lo == top_lo;
      any |= top_lo;
    } else {
      any = __reduce_max_sync(~0u, (unsigned)best);
      cand = (unsigned)best == any;
    }
    if (any == 0u) break;                                  // no expert is left
    const unsigned e = __reduce_min_sync(~0u, cand ? (unsigned)(at * 32 + lane) : ~0u);
    if (lane == r) chosen = (int)e;
    if (cand && (unsigned)(at * 32 + lane) == e) {
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (j == at) key[j] = 0ull;
    }
  }

  double s = 0.0;
  if (chosen >= 0) {
    const float xe = logit<T>(a.x, t * a.ld + chosen);
    s = a.softmax ? weight_of(xe, top) / total : sigmoid64(xe);
  }
  if (a.renorm) {
    const double sum = warp_sum64(s);
    s = sum > 0.0 ? s / sum : 0.0;
  }
  if (lane < a.topk) {
    a.idx[t * a.topk + lane] = chosen;
    a.p[t * a.topk + lane] = (float)(s * a.factor);
  }
}

template <typename T, int EPL>
cudaError_t launch_route_epl(const RouteArgs& a, bool scored, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.rows + kWarps - 1) / kWarps);
  const size_t smem = a.groups > 1 ? sizeof(double) * kWarps * EPL * 32 : 0;
  if (scored) return launch_pdl(expert_route_kernel<T, EPL, true>, dim3(grid), dim3(kWarps * 32), smem, st, a);
  return launch_pdl(expert_route_kernel<T, EPL, false>, dim3(grid), dim3(kWarps * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_route(const RouteArgs& a, bool scored, cudaStream_t st) {
  const int epl = (a.E + 31) / 32;
  if (epl <= 1) return launch_route_epl<T, 1>(a, scored, st);
  if (epl <= 2) return launch_route_epl<T, 2>(a, scored, st);
  if (epl <= 4) return launch_route_epl<T, 4>(a, scored, st);
  if (epl <= 8) return launch_route_epl<T, 8>(a, scored, st);
  if (epl <= 16) return launch_route_epl<T, 16>(a, scored, st);
  return launch_route_epl<T, 32>(a, scored, st);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_route_dev(const void* logits, long long ld, int dtype, int rows, int E, const float* bias, int score,
                             int n_group, int keep_group, int group_top, int top_k, int renorm, double factor,
                             int* topk_idx, float* topk_p, void* stream) {
  static const char who[] = "moe_route_dev";
  if (!at::elem_size(dtype)) return at::fail(MOE_ERR_INVALID, "%s: dtype %d (f32, f16 or bf16 is wanted)", who, dtype);
  if (rows < 0 || E < 1 || ld < E) return at::fail(MOE_ERR_INVALID, "%s: rows %d, E %d, ld %lld", who, rows, E, ld);
  if (E > 1024) return at::fail(MOE_ERR_UNSUPPORTED, "%s: %d experts (at most 1024)", who, E);
  if (score != MOE_ROUTE_SOFTMAX && score != MOE_ROUTE_SIGMOID) return at::fail(MOE_ERR_INVALID, "%s: score %d", who, score);
  if (n_group < 1 || E % n_group || keep_group < 1 || keep_group > n_group)
    return at::fail(MOE_ERR_INVALID, "%s: %d of %d groups over %d experts", who, keep_group, n_group, E);
  if (n_group > 32) return at::fail(MOE_ERR_UNSUPPORTED, "%s: %d groups (at most 32)", who, n_group);
  if (group_top != 1 && group_top != 2) return at::fail(MOE_ERR_INVALID, "%s: group_top %d (1 or 2)", who, group_top);
  if (top_k < 1 || top_k > keep_group * (E / n_group))
    return at::fail(MOE_ERR_INVALID, "%s: top %d of %d experts", who, top_k, keep_group * (E / n_group));
  if (top_k > 32) return at::fail(MOE_ERR_UNSUPPORTED, "%s: top %d (at most 32)", who, top_k);
  if (rows == 0) return MOE_OK;
  if (!logits || !topk_idx || !topk_p) return at::fail(MOE_ERR_INVALID, "%s: logits, topk_idx and topk_p are needed", who);
  at::OnDeviceOf on;
  int rc = on.enter(logits, who);
  if (rc) return rc;
  RouteArgs a{};
  a.x = logits; a.bias = bias; a.idx = topk_idx; a.p = topk_p; a.ld = ld; a.rows = rows; a.E = E;
  a.softmax = score == MOE_ROUTE_SOFTMAX; a.groups = keep_group == n_group ? 1 : n_group; a.keep = keep_group;
  a.group_top = group_top; a.topk = top_k; a.renorm = renorm != 0; a.factor = factor; a.group_size = E / n_group;
  a.lanes_per_group = 1;
  while (2 * a.lanes_per_group * n_group <= 32) a.lanes_per_group *= 2;
  const bool scored = bias || a.groups > 1;
  cudaStream_t st = (cudaStream_t)stream;
  return at::launched(dtype == MOE_DTYPE_F32    ? launch_route<float>(a, scored, st)
                      : dtype == MOE_DTYPE_BF16 ? launch_route<__nv_bfloat16>(a, scored, st)
                                                : launch_route<__half>(a, scored, st), who);
}
