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
// The choice is an ordering, and it is the order of the exact scores that is
// wanted: in fp32 two different sigmoid scores near 1 (or scores plus a bias)
// round to the same number often enough to change which expert is chosen.
// Without a bias the order of the scores is the order of the logits, exactly,
// and the experts (with groups: those of the groups that stay) are taken by
// logit. (Scores, even in 64 bits, would not do: the sigmoid is 1 from 37 on.)
// With a bias a token is first ranked by fp32 choices, whose error is bounded
// (`margin`): the list of the best goes on past top_k until the next is clearly
// behind, and if two neighbours in it are closer than the bound, its few experts
// are ordered again by choices in 64 bits. Groups are chosen by fp32 sums too,
// and where their bounds meet across the cut, by sums in 64 bits.
// The weights are fp32 softmax or sigmoid values.
//
// One warp routes one token: expert j * 32 + lane in lane `lane`. A round of
// the selection takes the largest key by a warp reduction, then the lowest
// index that has it by another; 16-bit logits carry the index in the key's
// other half and need one. Its logits are a few hundred bytes; the bound is
// instructions: issue slots where tokens are many (16384 of 128 experts: 77 %
// of them busy), the chain of one warp where they are less than a wave (4096 of
// 256 with groups and bias: 48 % busy, 36 % of the warps active, 9.8 us).
#include "attn.cuh"

#include <type_traits>

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
  at::FastDiv group;
  float factor;
};

// order-preserving keys; 0 is below every number's key, and -0 and 0 are one
__device__ __forceinline__ unsigned long long key_of(double c) {
  const long long b = __double_as_longlong(c + 0.0);
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ unsigned key_of(float c) {
  const int b = __float_as_int(c + 0.0f);
  return (unsigned)b ^ (b < 0 ? ~0u : 1u << 31);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key >> 31 ? key ^ (1u << 31) : ~key);
}
template <typename F> __device__ __forceinline__ F warp_sum_of(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

template <typename T> __device__ __forceinline__ float logit(const void* x, long long i);
template <> __device__ __forceinline__ float logit<float>(const void* x, long long i) { return ((const float*)x)[i]; }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(const void* x, long long i) { return __bfloat162float(((const __nv_bfloat16*)x)[i]); }
template <> __device__ __forceinline__ float logit<__half>(const void* x, long long i) { return __half2float(((const __half*)x)[i]); }

// exp(x - top) with x = top = +inf counted as 1, and the sigmoid: for the
// weights, in 64 bits, and (fast_) for the fp32 ranking, by the hardware's base-2
// exponential (2^-22) and reciprocal (1 ulp).
__device__ __forceinline__ float soft(float x, float top) { return x == top ? 1.0f : expf(x - top); }
__device__ __forceinline__ float sigm(float x) { return 1.0f / (1.0f + expf(-x)); }
__device__ __forceinline__ double soft64(float x, float top) { return x == top ? 1.0 : exp((double)x - (double)top); }
__device__ __forceinline__ double sigm64(float x) { return 1.0 / (1.0 + exp(-(double)x)); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_soft(float x, float top) { return x == top ? 1.0f : ex2((x - top) * 1.4426950408889634f); }
__device__ __forceinline__ float fast_sigm(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(x * -1.4426950408889634f)));
  return r;
}

// Scores plus bias of a lane's experts, in F; -inf for an expert that may not
// be chosen (a NaN or -inf logit or bias).
template <typename F, int EPL>
__device__ __forceinline__ void choices(const RouteArgs& a, const float (&x)[EPL], float top, F (&c)[EPL]) {
  const int lane = threadIdx.x & 31;
  F sum = 0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    if constexpr (sizeof(F) == 8) c[j] = a.softmax ? soft64(x[j], top) : sigm64(x[j]);
    else c[j] = a.softmax ? fast_soft(x[j], top) : fast_sigm(x[j]);
    if (!(x[j] > -INFINITY)) c[j] = 0;
    sum += c[j];
  }
  if (a.softmax) {
    sum = warp_sum_of(sum);
    if constexpr (sizeof(F) == 8) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) c[j] = c[j] / sum;
    } else {
      const float inv = 1.0f / sum;
#pragma unroll
      for (int j = 0; j < EPL; ++j) c[j] *= inv;
    }
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    if (a.bias && j * 32 + lane < a.E) c[j] += (F)a.bias[j * 32 + lane];
    if (!(x[j] > -INFINITY && c[j] > -INFINITY)) c[j] = -INFINITY;
  }
}

// How far apart two fp32 choices must be for the exact ones to be ordered
// alike. In units of 2^-24: a sigmoid errs by 6 (the exponential by 4 and its
// argument's rounding, both damped by e^-x s^2 < 1/4 and |x| e^-x s^2 < 1/2; the
// sum by 1, the reciprocal by 2), with the bias by |c| more, two of them by less
// than 2^4 (1 + |u| + |v|); a softmax score relatively by 2 |z| (its argument
// z = x - max, rounded twice; |z| s < 0.4), 4 (the exponential), 2 (quotient and
// product) and by its sum, up to 37 roundings, 4 and twice the mean of |z|,
// below ln 1024 + 1: less than 2^6, two of them and the bias 2^7 (1 + |u| + |v|).
// `drop`: the low bits of either that were taken out, relatively 2^(drop - 23).
__device__ __forceinline__ float margin(const RouteArgs& a, float u, float v, float drop) {
  const float m = fabsf(u) + fabsf(v);
  return fmaf(m, drop, (a.softmax ? 0x1p-17f : 0x1p-20f) * (1.0f + m));
}

// Which of the groups stay, a bit at lane (group * lanes_per_group). sure (fp32):
// whether 64-bit sums choose the same. A group's sum errs by no more than the
// margin of its two addends (which may be large and cancel; the sum's own
// rounding is below what the margin has to spare), so it is sure where no
// group that stays may lie below one that does not.
template <typename F, int EPL>
__device__ __forceinline__ unsigned best_groups(const RouteArgs& a, F* mine, const F (&c)[EPL], bool& sure) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < EPL; ++j) mine[j * 32 + lane] = c[j];
  __syncwarp();
  // lanes_per_group lanes look through a group and merge their best two
  const int lpg = a.lanes_per_group, grp = lane / lpg;
  F b0 = -INFINITY, b1 = -INFINITY;
  if (grp < a.groups)
    for (int i = lane % lpg; i < a.group_size; i += lpg) {
      const F v = mine[grp * a.group_size + i];
      b1 = max(b1, min(b0, v));
      b0 = max(b0, v);
    }
  for (int o = 1; o < lpg; o <<= 1) {
    const F o0 = __shfl_xor_sync(~0u, b0, o), o1 = __shfl_xor_sync(~0u, b1, o);
    b1 = max(min(b0, o0), max(b1, o1));
    b0 = max(b0, o0);
  }
  const F second = a.group_top == 2 && b1 > -INFINITY ? b1 : (F)0, gs = b0 + second;
  // a group stays if fewer than `keep` groups come before it
  int before = 0;
  for (int h = 0; h < a.groups; ++h) {
    const F v = __shfl_sync(~0u, gs, h * lpg);
    before += v > gs || (v == gs && h < grp);
  }
  const bool head = grp < a.groups && lane % lpg == 0, stays = head && before < a.keep;
  if constexpr (sizeof(F) == 4) {
    const float e = b0 > -INFINITY ? margin(a, b0, second, 0.f) : 0.f;     // a group without experts is exact
    const unsigned least = __reduce_min_sync(~0u, stays ? key_of(gs - e) : ~0u);
    const unsigned most = __reduce_max_sync(~0u, head && !stays ? key_of(gs + e) : 0u);
    sure = !__any_sync(~0u, head && !(e < INFINITY)) && least >= most;
  }
  return __ballot_sync(~0u, stays);
}

// The same by choices in 64 bits.
template <int EPL>
__device__ __noinline__ unsigned best_groups64(const RouteArgs& a, const float (&x)[EPL], float top, double* mine) {
  double c[EPL];
  bool sure;
  choices<double, EPL>(a, x, top, c);
  return best_groups<double, EPL>(a, mine, c, sure);
}

// Whether expert j * 32 + lane is in a group that stays.
__device__ __forceinline__ bool stays_in(const RouteArgs& a, unsigned stays, int j) {
  const int e = j * 32 + (threadIdx.x & 31);
  return e >= a.E || (stays >> ((int)a.group.div((unsigned)e) * a.lanes_per_group)) & 1;
}

// Keys of a lane, the largest first (odd-even exchange; EPL is a power of two).
template <int EPL>
__device__ __forceinline__ void sort_keys(unsigned (&k)[EPL]) {
#pragma unroll
  for (int p = 1; p < EPL; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < EPL; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (j + i + q < EPL && (j + i) / (2 * p) == (j + i + q) / (2 * p)) {
            const unsigned u = k[j + i], v = k[j + i + q];
            k[j + i] = max(u, v);
            k[j + i + q] = min(u, v);
          }
}
// One round over sorted unique keys: the largest of the warp leaves its lane.
template <int EPL>
__device__ __forceinline__ unsigned pop(unsigned (&k)[EPL]) {
  const unsigned best = __reduce_max_sync(~0u, k[0]);
  const bool own = k[0] == best;
#pragma unroll
  for (int j = 0; j + 1 < EPL; ++j) k[j] = own ? k[j + 1] : k[j];
  if (own) k[EPL - 1] = 0u;
  return best;
}

// One round: the largest of the warp's keys, the lowest expert that has it
// (which then leaves), or -1.
template <int EPL>
__device__ __forceinline__ int take(unsigned (&key)[EPL], unsigned& top) {
  const int lane = threadIdx.x & 31;
  unsigned best = key[0];
  int at = 0;
#pragma unroll
  for (int j = 1; j < EPL; ++j)
    if (key[j] > best) { best = key[j]; at = j; }
  top = __reduce_max_sync(~0u, best);
  if (top == 0u) return -1;
  const unsigned mine = at * 32 + lane, e = __reduce_min_sync(~0u, best == top ? mine : ~0u);
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    if (j * 32 + lane == e) key[j] = 0u;
  return (int)e;
}
template <int EPL>
__device__ __forceinline__ int take(unsigned long long (&key)[EPL]) {
  const int lane = threadIdx.x & 31;
  unsigned long long best = key[0];
  int at = 0;
#pragma unroll
  for (int j = 1; j < EPL; ++j)
    if (key[j] > best) { best = key[j]; at = j; }
  const unsigned hi = (unsigned)(best >> 32), top_hi = __reduce_max_sync(~0u, hi);
  const unsigned lo = hi == top_hi ? (unsigned)best : 0u, top_lo = __reduce_max_sync(~0u, lo);
  if ((top_hi | top_lo) == 0u) return -1;
  const bool cand = hi == top_hi && lo == top_lo;
  const unsigned mine = at * 32 + lane, e = __reduce_min_sync(~0u, cand ? mine : ~0u);
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    if (j * 32 + lane == e) key[j] = 0ull;
  return (int)e;
}

// The token's choice ranked in 64 bits; lane r returns the r-th.
template <int EPL>
__device__ __noinline__ int choose64(const RouteArgs& a, const float (&x)[EPL], float top, unsigned stays) {
  double c[EPL];
  unsigned long long key[EPL];
  choices<double, EPL>(a, x, top, c);
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    key[j] = c[j] > -INFINITY && (a.groups == 1 || stays_in(a, stays, j)) ? key_of(c[j]) : 0ull;
  int chosen = -1;
  for (int r = 0; r < a.topk; ++r) {
    const int e = take<EPL>(key);
    if (e < 0) break;
    if ((threadIdx.x & 31) == r) chosen = e;
  }
  return chosen;
}

// With a bias: the n experts that lanes 0 .. n - 1 list, in the order of their
// choices in 64 bits; lane r returns the r-th.
template <typename T, int EPL>
__device__ __noinline__ int order64(const RouteArgs& a, const float (&x)[EPL], float top, long long t, int listed, int n) {
  const int lane = threadIdx.x & 31;
  double total = 1.0;
  if (a.softmax) {
    total = 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) total += x[j] > -INFINITY ? soft64(x[j], top) : 0.0;
    total = warp_sum_of(total);
  }
  double c = 0.0;
  if (lane < n) {
    const float xe = logit<T>(a.x, t * a.ld + listed);
    c = (a.softmax ? soft64(xe, top) / total : sigm64(xe)) + (double)a.bias[listed];
  }
  int rank = 0;
  for (int m = 0; m < n; ++m) {
    const double v = __shfl_sync(~0u, c, m);
    const int e = __shfl_sync(~0u, listed, m);
    rank += v > c || (v == c && e < listed);
  }
  int chosen = -1;
  for (int m = 0; m < n; ++m) {
    const int r = __shfl_sync(~0u, rank, m), e = __shfl_sync(~0u, listed, m);
    if (r == lane) chosen = e;
  }
  return chosen;
}

// The experts that stay, by logit; lane r returns the r-th.
template <typename T, int EPL>
__device__ __forceinline__ int choose_by_logit(const RouteArgs& a, const float (&x)[EPL], unsigned stays) {
  const int lane = threadIdx.x & 31;
  unsigned key[EPL];
  int chosen = -1;
  if constexpr (sizeof(T) == 2) {
    // the logit's 16 bits above, the index from the top down below them
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const unsigned e = j * 32 + lane;
      unsigned b;
      if constexpr (std::is_same<T, __half>::value) b = __half_as_ushort(__float2half_rn(x[j] + 0.0f));
      else b = __float_as_uint(x[j] + 0.0f) >> 16;
      b = (b ^ (b >> 15 ? 0xffffu : 0x8000u)) & 0xffffu;
      key[j] = x[j] > -INFINITY && (stays == ~0u || stays_in(a, stays, j)) ? b << 16 | (0xffffu - e) : 0u;
    }
    sort_keys<EPL>(key);
    unsigned mine = 0u;
    for (int r = 0; r < a.topk; ++r) {
      const unsigned best = pop<EPL>(key);
      if (best == 0u) break;
      if (lane == r) mine = best;
    }
    chosen = mine ? 0xffff - (int)(mine & 0xffffu) : -1;
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      key[j] = x[j] > -INFINITY && (stays == ~0u || stays_in(a, stays, j)) ? key_of(x[j]) : 0u;
    for (int r = 0; r < a.topk; ++r) {
      unsigned k;
      const int e = take<EPL>(key, k);
      if (e < 0) break;
      if (lane == r) chosen = e;
    }
  }
  return chosen;
}

// EPL experts a lane. MODE: what the choice needs: logits alone; every score for
// the groups, then logits; every score and the bias.
enum { kByLogit, kByGroup, kByScore };
template <typename T, int EPL, int MODE>
__global__ void __launch_bounds__(kWarps * 32) expert_route_kernel(const RouteArgs a) {
  extern __shared__ double choice_sm[];                    // groups: [kWarps][EPL * 32]
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = (long long)blockIdx.x * kWarps + warp;
  if (t >= a.rows) return;
  float x[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = j * 32 + lane;
    x[j] = e < a.E ? logit<T>(a.x, t * a.ld + e) : -INFINITY;
    if (!(x[j] > -INFINITY)) x[j] = -INFINITY;            // NaN: never chosen, as -inf
  }
  float top = -INFINITY;
  int chosen = -1;                                         // lane r: the r-th choice
  if constexpr (MODE != kByLogit) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) top = fmaxf(top, x[j]);
    const unsigned tk = __reduce_max_sync(~0u, key_of(top));
    top = value_of(tk);
    float c[EPL];
    choices<float, EPL>(a, x, top, c);
    unsigned stays = ~0u;
    if (a.groups > 1) {
      double* mine = choice_sm + warp * (EPL * 32);
      bool sure;
      stays = best_groups<float, EPL>(a, (float*)mine, c, sure);
      if (!sure) stays = best_groups64<EPL>(a, x, top, mine);
      if constexpr (MODE == kByScore)
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (!stays_in(a, stays, j)) c[j] = -INFINITY;
    }
    if constexpr (MODE == kByGroup) {
      chosen = choose_by_logit<T, EPL>(a, x, stays);
    } else {
      // Keys: the fp32 choice without its lowest bits, which hold the index from
      // the top down. Lane n keeps the n-th; top_k + 1 of them, and on until the
      // next one is clearly behind the one before: nothing outside the list can
      // then belong in its first top_k.
      constexpr unsigned kLow = EPL * 32 - 1;
      constexpr float kDrop = (float)(EPL * 32) * 0x1p-23f;
      unsigned key[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        key[j] = c[j] > -INFINITY ? (key_of(c[j]) & ~kLow) | (kLow - (j * 32 + lane)) : 0u;
      sort_keys<EPL>(key);
      unsigned mine = 0u;
      int n = 0;
      for (; n < min(a.topk + 1, 32); ++n) {
        const unsigned best = pop<EPL>(key);
        if (best == 0u) break;
        if (lane == n) mine = best;
      }
      auto near = [&]() -> unsigned {                        // bit i: entry i + 1 is not clearly behind entry i
        const float u = value_of(mine & ~kLow), v = __shfl_down_sync(~0u, u, 1);
        return __ballot_sync(~0u, lane + 1 < n && !(u - v >= margin(a, u, v, kDrop)));
      };
      unsigned close = near();
      bool anew = false;
      while (n > a.topk && (close >> (n - 2)) & 1) {         // the last is not: the list goes on
        const unsigned best = pop<EPL>(key);
        if (best == 0u) break;
        if (n == 32) { anew = true; break; }
        if (lane == n) mine = best;
        ++n;
        close = near();
      }
      if (a.topk == 32 && !anew) {                           // no lane is left to look behind the last
        const unsigned best = pop<EPL>(key);
        const float u = __shfl_sync(~0u, value_of(mine & ~kLow), 31), v = value_of(best & ~kLow);
        anew = best != 0u && !(u - v >= margin(a, u, v, kDrop));
      }
      chosen = mine ? (int)(kLow - (mine & kLow)) : -1;
      if (anew) chosen = choose64<EPL>(a, x, top, stays);
      else if (close) chosen = order64<T, EPL>(a, x, top, t, chosen, __popc(__ballot_sync(~0u, mine != 0u)));
      if (lane >= a.topk) chosen = -1;
    }
  } else {
    chosen = choose_by_logit<T, EPL>(a, x, ~0u);
  }

  const float xe = chosen >= 0 ? logit<T>(a.x, t * a.ld + chosen) : 0.f;
  float s;
  if (a.renorm) {
    // only ratios matter: from the largest chosen logit, so that they survive
    // where the scores themselves would underflow (the sigmoid is
    // exp(x) / (1 + exp(x)))
    const float m = value_of(__reduce_max_sync(~0u, chosen >= 0 ? key_of(xe) : 0u));
    s = a.softmax ? soft(xe, m) : m > 0.f ? sigm(xe) : soft(xe, m) / (1.0f + expf(xe));
    if (chosen < 0) s = 0.f;
    const float sum = warp_sum_of(s);
    s = sum > 0.f ? s / sum : 0.f;
  } else if (a.softmax) {
    if constexpr (MODE == kByLogit) top = __shfl_sync(~0u, xe, 0);  // the first choice is the largest logit
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) sum += x[j] > -INFINITY ? soft(x[j], top) : 0.f;
    sum = warp_sum_of(sum);
    s = chosen >= 0 ? soft(xe, top) / sum : 0.f;
  } else {
    s = chosen >= 0 ? sigm(xe) : 0.f;
  }
  if (lane < a.topk) {
    a.idx[t * a.topk + lane] = chosen;
    a.p[t * a.topk + lane] = s * a.factor;
  }
}

template <typename T, int EPL>
cudaError_t launch_route_epl(const RouteArgs& a, cudaStream_t st) {
  const unsigned grid = ((unsigned)a.rows + kWarps - 1) / kWarps;
  const size_t smem = a.groups > 1 ? sizeof(double) * kWarps * EPL * 32 : 0;
  if (a.bias) return launch_pdl(expert_route_kernel<T, EPL, kByScore>, dim3(grid), dim3(kWarps * 32), smem, st, a);
  if (a.groups > 1) return launch_pdl(expert_route_kernel<T, EPL, kByGroup>, dim3(grid), dim3(kWarps * 32), smem, st, a);
  return launch_pdl(expert_route_kernel<T, EPL, kByLogit>, dim3(grid), dim3(kWarps * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_route(const RouteArgs& a, cudaStream_t st) {
  const int epl = (a.E + 31) / 32;
  if (epl <= 1) return launch_route_epl<T, 1>(a, st);
  if (epl <= 2) return launch_route_epl<T, 2>(a, st);
  if (epl <= 4) return launch_route_epl<T, 4>(a, st);
  if (epl <= 8) return launch_route_epl<T, 8>(a, st);
  if (epl <= 16) return launch_route_epl<T, 16>(a, st);
  return launch_route_epl<T, 32>(a, st);
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
  a.group_top = group_top; a.topk = top_k; a.renorm = renorm != 0; a.factor = (float)factor; a.group_size = E / n_group;
  a.group = at::FastDiv((unsigned)(E / n_group));
  a.lanes_per_group = 1;
  while (2 * a.lanes_per_group * n_group <= 32) a.lanes_per_group *= 2;
  cudaStream_t st = (cudaStream_t)stream;
  return at::launched(dtype == MOE_DTYPE_F32    ? launch_route<float>(a, st)
                      : dtype == MOE_DTYPE_BF16 ? launch_route<__nv_bfloat16>(a, st)
                                                : launch_route<__half>(a, st), who);
}
