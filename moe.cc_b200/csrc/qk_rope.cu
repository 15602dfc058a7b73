// qk_rope.cu — moe_qk_norm_rope_dev: RMSNorm of every query and key head, the
// position rotation, and the append of K and V to the paged cache, in one pass
// over the new rows (test_model_trace.c:357-392 does the same in separate loops
// on the CPU).
//
//   y = x / sqrt(mean(x^2) + eps) * w                       per head
//   (y_i, y_{i+R/2}) <- (y_i c_i - y_{i+R/2} s_i, y_{i+R/2} c_i + y_i s_i),  i < R/2
//
// with (c, s) = row `position` of the caller's table and R the rotated width;
// elements from R on pass through. All of it in fp32, each output rounded once.
//
// The bound is bytes: every element is read once and written once, so the rest
// has to stay small. A head is held by LPH lanes, each with a run of R elements
// of the lower half and the R that rotate with them from the upper half: the
// rotation needs no exchange between lanes and the mean is a shuffle sum. Norm
// weight and rotation are one pair of factors,
//   y_lo = inv (x_lo (w_lo c) - x_hi (w_hi s)),  y_hi = inv (x_hi (w_hi c) + x_lo (w_lo s)),
// which a warp works out once for its row and applies to all the heads that it
// takes of it: all of them in a long batch, 32 / LPH where rows are few.
#include "attn.cuh"

namespace moe {
namespace {

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *kc, *vc;
  const float *q_norm, *k_norm, *rope;
  const int *row_pos, *row_slot;
  long long ldq, ldk, ldv, ldo, page_stride, token_stride, head_stride;
  int rows, n_q, n_kv, hd, rot, rope_len, n_slots, page_size;
  int per_row;            // warps a row
  float eps;
  at::FastDiv page;
};

constexpr int kWarps = 4;

// R consecutive elements in one or two 16-byte (R = 4 of 16 bits: 8-byte) pieces
template <typename T, int R> struct Run {
  typename at::Vec4<T>::raw v[R / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 2 && R == 8) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    else
#pragma unroll
      for (int i = 0; i < R / 4; ++i) v[i] = reinterpret_cast<const typename at::Vec4<T>::raw*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) == 2 && R == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    else
#pragma unroll
      for (int i = 0; i < R / 4; ++i) reinterpret_cast<typename at::Vec4<T>::raw*>(p)[i] = v[i];
  }
  __device__ __forceinline__ void get(float (&f)[R]) const {
#pragma unroll
    for (int i = 0; i < R / 4; ++i) at::Vec4<T>::get(v[i], f + 4 * i);
  }
  __device__ __forceinline__ void put(const float (&f)[R]) {
#pragma unroll
    for (int i = 0; i < R / 4; ++i) v[i] = at::Vec4<T>::put(f + 4 * i);
  }
};

// Heads `first`, `first` + step, ... of one row's queries or keys, a warp's
// 32 / LPH at a time.
template <typename TI, typename TO, int R, int LPH>
__device__ __forceinline__ void turn_heads(const RopeArgs& a, const TI* src, TO* dst, long long dst_stride, int heads,
                                           const float* w, int first, int step, int lo, int hi, bool on, bool turns,
                                           const float (&c)[R], const float (&s)[R]) {
  constexpr int kHeads = 32 / LPH;
  if (first * kHeads >= heads) return;
  const int g = (threadIdx.x & 31) / LPH;
  float lc[R], ls[R], hc[R], hs[R];       // w_lo c, w_lo s, w_hi c, w_hi s
#pragma unroll
  for (int i = 0; i < R; ++i) { lc[i] = hc[i] = c[i]; ls[i] = hs[i] = s[i]; }
  if (w && on) {
    Run<float, R> wl, wh;
    float l[R], h[R];
    wl.load(w + lo); wh.load(w + hi);
    wl.get(l); wh.get(h);
#pragma unroll
    for (int i = 0; i < R; ++i) { lc[i] *= l[i]; ls[i] *= l[i]; hc[i] *= h[i]; hs[i] *= h[i]; }
  }
  const float inv_hd = 1.0f / (float)a.hd;
  Run<TI, R> xl, xh;
  auto fetch = [&](int t) {
    const int h = t * kHeads + g;
    if (on && h < heads) { xl.load(src + (long long)h * a.hd + lo); xh.load(src + (long long)h * a.hd + hi); }
  };
  fetch(first);
  for (int t = first; t * kHeads < heads; t += step) {
    float x[R] = {}, y[R] = {};
    const int h = t * kHeads + g;
    const bool live = on && h < heads;
    if (live) { xl.get(x); xh.get(y); }
    fetch(t + step);                       // the next heads are on their way meanwhile
    float inv = 1.0f;
    if (w) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) sq = fmaf(x[i], x[i], fmaf(y[i], y[i], sq));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
      inv = rsqrtf(fmaf(sq, inv_hd, a.eps));
    }
    if (!live) continue;
    if (turns) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float e = x[i], o = y[i];
        x[i] = (e * lc[i] - o * hs[i]) * inv;
        y[i] = (o * hc[i] + e * ls[i]) * inv;
      }
    } else if (w) {
#pragma unroll
      for (int i = 0; i < R; ++i) { x[i] *= lc[i] * inv; y[i] *= hc[i] * inv; }
    }
    Run<TO, R> out;
    out.put(x);
    out.store(dst + h * dst_stride + lo);
    out.put(y);
    out.store(dst + h * dst_stride + hi);
  }
}

template <typename TI, typename TO, int R, int LPH>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_rope_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch();
  constexpr int kHeads = 32 / LPH;
  // warp `first` of `step` on this row
  const long long id = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int row = (int)(id / a.per_row), first = (int)(id % a.per_row), step = a.per_row;
  if (row >= a.rows) return;
  const int l = threadIdx.x % LPH;
  const int pos = a.row_pos ? a.row_pos[row] : 0;
  const int slot = a.row_slot ? a.row_slot[row] : -1;
  if (pos < 0 || (a.rot && pos >= a.rope_len)) return;      // a padded row: nothing of it is touched
  const bool on = R * l < a.hd / 2;
  // this lane's pairs (lo + i, hi + i)
  int lo = R * l, hi = R * l + a.rot / 2;
  const bool turns = lo < a.rot / 2;
  if (!turns) { lo = R * l + a.rot / 2; hi = lo + (a.hd - a.rot) / 2; }
  float c[R], s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) { c[i] = 1.f; s[i] = 0.f; }
  if (on && turns) {
    const float* t = a.rope + (long long)pos * a.rot + lo;
    Run<float, R> v;
    v.load(t); v.get(c);
    v.load(t + a.rot / 2); v.get(s);
  }
  turn_heads<TI, TO, R, LPH>(a, (const TI*)a.q + row * a.ldq, (TO*)a.q_out + row * a.ldo, a.hd, a.n_q, a.q_norm, first, step,
                             lo, hi, on, turns, c, s);
  if (slot < 0 || slot >= a.n_slots) return;
  const int pg = (int)a.page.div((unsigned)slot);
  const long long to = pg * a.page_stride + (slot - pg * a.page_size) * a.token_stride;
  // the groups of heads are dealt to the row's warps queries first, then keys, then values
  const int nq = (a.n_q + kHeads - 1) / kHeads, nk = (a.n_kv + kHeads - 1) / kHeads;
  const int fk = (first - nq % step + step) % step, fv = (fk - nk % step + step) % step;
  turn_heads<TI, TO, R, LPH>(a, (const TI*)a.k + row * a.ldk, (TO*)a.kc + to, a.head_stride, a.n_kv, a.k_norm, fk, step,
                             lo, hi, on, turns, c, s);
  const int g = (threadIdx.x & 31) / LPH;
  const TI* v = (const TI*)a.v + row * a.ldv;
  for (int h = fv * kHeads + g; h < a.n_kv; h += step * kHeads) {
    if (!on) continue;
    Run<TI, R> xl, xh;
    xl.load(v + (long long)h * a.hd + lo);
    xh.load(v + (long long)h * a.hd + hi);
    TO* dst = (TO*)a.vc + to + h * a.head_stride;
    if constexpr (sizeof(TI) == sizeof(TO)) {
      xl.store((TI*)(dst + lo));
      xh.store((TI*)(dst + hi));
    } else {
      Run<TO, R> out;
      float x[R];
      xl.get(x); out.put(x); out.store(dst + lo);
      xh.get(x); out.put(x); out.store(dst + hi);
    }
  }
}

template <typename TI, typename TO>
cudaError_t launch_rope(RopeArgs a, cudaStream_t st) {
  auto go = [&](auto kernel, int lph) {
    // One warp a row where that fills the GPU (16 warps an SM), else as many
    // as the row has groups of heads
    const int per = 32 / lph, groups = (a.n_q + per - 1) / per + 2 * ((a.n_kv + per - 1) / per);
    const long long want = (2368 + a.rows - 1) / a.rows;
    a.per_row = (int)(want < groups ? want : groups);
    const long long blocks = ((long long)a.rows * a.per_row + kWarps - 1) / kWarps;
    return launch_pdl(kernel, dim3((unsigned)blocks), dim3(kWarps * 32), 0, st, a);
  };
  // runs of 8 where the halves of what rotates and of what does not are whole
  // numbers of them
  if (a.rot % 16 == 0 && (a.hd - a.rot) % 16 == 0) {
    if (a.hd <= 64) return go(qk_norm_rope_kernel<TI, TO, 8, 4>, 4);
    if (a.hd <= 128) return go(qk_norm_rope_kernel<TI, TO, 8, 8>, 8);
    return go(qk_norm_rope_kernel<TI, TO, 8, 16>, 16);
  }
  if (a.hd <= 64) return go(qk_norm_rope_kernel<TI, TO, 4, 8>, 8);
  if (a.hd <= 128) return go(qk_norm_rope_kernel<TI, TO, 4, 16>, 16);
  return go(qk_norm_rope_kernel<TI, TO, 4, 32>, 32);
}

// whether the row-strided ranges [p, p + ((rows-1) ld + n) es) of two
// operands share a byte
bool overlap(const void* p, long long ldp, long long np, int ep, const void* r, long long ldr, long long nr, int er,
             int rows) {
  const uintptr_t p0 = (uintptr_t)p, p1 = p0 + (uintptr_t)(((rows - 1) * ldp + np) * ep);
  const uintptr_t r0 = (uintptr_t)r, r1 = r0 + (uintptr_t)(((rows - 1) * ldr + nr) * er);
  return p0 < r1 && r0 < p1;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_qk_norm_rope_dev(const void* q, long long ldq, const void* k, long long ldk, const void* v,
                                    long long ldv, int dtype, int rows, int n_q, const float* q_norm,
                                    const float* k_norm, float eps, const float* rope, int rot_dim, int rope_len,
                                    const int* row_pos, const int* row_slot, void* q_out, long long ldo,
                                    const MoeKvCache* cache, void* stream) {
  static const char who[] = "moe_qk_norm_rope_dev";
  int rc = at::check_cache(cache, who);
  if (rc) return rc;
  const int es = at::elem_size(dtype), eo = at::elem_size(cache->dtype), hd = cache->head_dim;
  if (!es) return at::fail(MOE_ERR_INVALID, "%s: dtype %d (f32, f16 or bf16 is wanted)", who, dtype);
  if (es == 2 && dtype != cache->dtype)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: 16-bit rows need a cache of their own type", who);
  if (rows < 0 || n_q < 0 || (long long)n_q + 2ll * cache->n_kv > 32768)
    return at::fail(MOE_ERR_INVALID, "%s: rows %d, n_q %d, n_kv %d", who, rows, n_q, cache->n_kv);
  if (n_q && (!q || !q_out)) return at::fail(MOE_ERR_INVALID, "%s: q and q_out are needed", who);
  if (row_slot && (!k || !v)) return at::fail(MOE_ERR_INVALID, "%s: row_slot without k and v", who);
  if (rot_dim < 0 || rot_dim > hd || rot_dim % 8)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: rot_dim %d (multiples of 8 up to head_dim %d)", who, rot_dim, hd);
  if (rot_dim && (!rope || rope_len < 1 || !row_pos))
    return at::fail(MOE_ERR_INVALID, "%s: a rotation needs rope, rope_len and row_pos", who);
  if (!(eps >= 0.f)) return at::fail(MOE_ERR_INVALID, "%s: eps must not be negative", who);
  const int qi = 16 / es, qo = 16 / eo;
  if (n_q && (ldq < (long long)n_q * hd || ldo < (long long)n_q * hd))
    return at::fail(MOE_ERR_INVALID, "%s: rows of q or q_out overlap", who);
  if (n_q && ((uintptr_t)q % 16 || (uintptr_t)q_out % 16 || ldq % qi || ldo % qo))
    return at::fail(MOE_ERR_INVALID, "%s: rows of q and q_out must start on 16-byte boundaries", who);
  if (row_slot && ((uintptr_t)k % 16 || (uintptr_t)v % 16 || ldk % qi || ldv % qi || ldk < 0 || ldv < 0))
    return at::fail(MOE_ERR_INVALID, "%s: rows of k and v must start on 16-byte boundaries", who);
  if ((uintptr_t)q_norm % 16 || (uintptr_t)k_norm % 16 || (rot_dim && (uintptr_t)rope % 16))
    return at::fail(MOE_ERR_INVALID, "%s: norm weights and rope must be 16-byte aligned", who);
  if (rows == 0 || (n_q == 0 && !row_slot)) return MOE_OK;
  // q_out may be q itself; any other overlap would be read after it was written
  const long long nq = (long long)n_q * hd, nk = (long long)cache->n_kv * hd;
  const bool same = q_out == q && ldo == ldq && es == eo;
  if (n_q && !same && overlap(q_out, ldo, nq, eo, q, ldq, nq, es, rows))
    return at::fail(MOE_ERR_INVALID, "%s: q_out overlaps q without being q", who);
  if (n_q && !same && row_slot &&
      (overlap(q_out, ldo, nq, eo, k, ldk, nk, es, rows) || overlap(q_out, ldo, nq, eo, v, ldv, nk, es, rows)))
    return at::fail(MOE_ERR_INVALID, "%s: q_out overlaps k or v", who);
  at::OnDeviceOf on;
  if ((rc = on.enter(n_q ? q : k, who))) return rc;
  RopeArgs a{};
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kc = cache->k; a.vc = cache->v;
  a.q_norm = q_norm; a.k_norm = k_norm; a.rope = rope; a.row_pos = row_pos; a.row_slot = row_slot;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
  a.page_stride = cache->page_stride; a.token_stride = cache->token_stride; a.head_stride = cache->head_stride;
  a.rows = rows; a.n_q = n_q; a.n_kv = cache->n_kv; a.hd = hd; a.rot = rot_dim; a.rope_len = rope_len;
  a.n_slots = cache->n_pages * cache->page_size; a.page_size = cache->page_size; a.eps = eps;
  a.page = at::FastDiv((unsigned)cache->page_size);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == MOE_DTYPE_BF16) e = launch_rope<__nv_bfloat16, __nv_bfloat16>(a, st);
  else if (dtype == MOE_DTYPE_F16) e = launch_rope<__half, __half>(a, st);
  else if (cache->dtype == MOE_DTYPE_F32) e = launch_rope<float, float>(a, st);
  else if (cache->dtype == MOE_DTYPE_BF16) e = launch_rope<float, __nv_bfloat16>(a, st);
  else e = launch_rope<float, __half>(a, st);
  return at::launched(e, who);
}
