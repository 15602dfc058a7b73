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

constexpr int kWarps = 2;

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

// Two fp32 operations an instruction.
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 pack(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack(F2 p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.v)); }
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// FULL: the lanes of a head hold it exactly, all of it rotated.
template <typename TI, typename TO, int R, int LPH, bool FULL>
__global__ void __launch_bounds__(kWarps * 32, 8) qk_norm_rope_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch();
  constexpr int kHeads = 32 / LPH;
  // groups of queries on their way or worked on (4096 16-bit rows: 2 groups
  // 19.2 us, 3 17.8, 4 17.7; 1001 fp32 rows: 7.3, 7.8, 9.4)
  constexpr int kDepth = sizeof(TI) == 2 ? 3 : 2;
  const long long id = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int row = (int)(id / a.per_row), step = a.per_row, me = (int)(id - (long long)row * step);
  if (row >= a.rows) return;
  const int hd = FULL ? 2 * R * LPH : a.hd, rot = FULL ? hd : a.rot;
  const int l = threadIdx.x % LPH, g = (threadIdx.x & 31) / LPH;
  const bool on = FULL || R * l < hd / 2, turns = FULL || R * l < rot / 2;
  // this lane's pairs (lo + i, hi + i)
  int lo = R * l, hi = R * l + rot / 2;
  if (!turns) { lo = R * l + rot / 2; hi = lo + (hd - rot) / 2; }
  if (!on) lo = hi = 0;

  // The row's groups of kHeads heads, values, keys and queries, are dealt to
  // its warps. The first of each are on their way before anything is known of
  // the row. A lane past the last head repeats the last one and stores nothing.
  const int nk = a.row_slot ? (a.n_kv + kHeads - 1) / kHeads : 0, nq = (a.n_q + kHeads - 1) / kHeads;
  const int fk = (me - nk % step + step) % step, fq = (me - 2 * nk % step + step) % step;
  struct Pair { Run<TI, R> lo, hi; };
  auto fetch = [&](const TI* base, int t, int heads) {
    Pair r;
    const TI* p = base + min(t * kHeads + g, heads - 1) * hd;
    r.lo.load(p + lo);
    r.hi.load(p + hi);
    return r;
  };
  const TI *qrow = (const TI*)a.q + row * a.ldq, *krow = (const TI*)a.k + row * a.ldk, *vrow = (const TI*)a.v + row * a.ldv;
  Pair pv, pk, pq[kDepth];
  if (me < nk) pv = fetch(vrow, me, a.n_kv);
  if (fk < nk) pk = fetch(krow, fk, a.n_kv);
#pragma unroll
  for (int i = 0; i < kDepth; ++i)
    if (fq + i * step < nq) pq[i] = fetch(qrow, fq + i * step, a.n_q);
  const int pos = a.row_pos ? a.row_pos[row] : 0;
  const int slot = a.row_slot ? a.row_slot[row] : -1;
  if (pos < 0 || (rot && pos >= a.rope_len)) return;        // a padded row: nothing of it is written
  const float* cs = a.rope + (turns ? (long long)pos * rot + lo : 0);

  F2 lc[R / 2], ls[R / 2], hc[R / 2], hs[R / 2];       // w_lo c, w_lo s, w_hi c, -w_hi s
  auto factors = [&](const float* w) {
    float c[R], s[R], u[R], v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) { c[i] = u[i] = v[i] = 1.f; s[i] = 0.f; }
    Run<float, R> f;
    if (turns) { f.load(cs); f.get(c); f.load(cs + rot / 2); f.get(s); }
    if (w) { f.load(w + lo); f.get(u); f.load(w + hi); f.get(v); }
#pragma unroll
    for (int i = 0; i < R; i += 2) {
      lc[i / 2] = pack(c[i] * u[i], c[i + 1] * u[i + 1]);
      ls[i / 2] = pack(s[i] * u[i], s[i + 1] * u[i + 1]);
      hc[i / 2] = pack(c[i] * v[i], c[i + 1] * v[i + 1]);
      hs[i / 2] = pack(-s[i] * v[i], -s[i + 1] * v[i + 1]);
    }
  };
  const float inv_hd = 1.0f / (float)hd;
  auto turn = [&](const Pair& r, const float* w, TO* dst, bool store) {
    float x[R], y[R];
    r.lo.get(x);
    r.hi.get(y);
    F2 X[R / 2], Y[R / 2];
#pragma unroll
    for (int i = 0; i < R; i += 2) { X[i / 2] = pack(x[i], x[i + 1]); Y[i / 2] = pack(y[i], y[i + 1]); }
    float inv = 1.0f;
    if (w) {
      F2 s = mul(X[0], X[0]);
#pragma unroll
      for (int i = 1; i < R / 2; ++i) s = fma(X[i], X[i], s);
#pragma unroll
      for (int i = 0; i < R / 2; ++i) s = fma(Y[i], Y[i], s);
      float s0, s1;
      unpack(s, s0, s1);
      float sq = on ? s0 + s1 : 0.f;
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
      inv = rsqrtf(fmaf(sq, inv_hd, a.eps));
    }
    if (!on || !store) return;
    if (turns || w) {
      const F2 n = pack(inv, inv);
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        F2 u = mul(X[i], lc[i]), v = mul(Y[i], hc[i]);
        if (turns) { u = fma(Y[i], hs[i], u); v = fma(X[i], ls[i], v); }
        unpack(mul(u, n), x[2 * i], x[2 * i + 1]);
        unpack(mul(v, n), y[2 * i], y[2 * i + 1]);
      }
    }
    Run<TO, R> out;
    out.put(x);
    out.store(dst + lo);
    out.put(y);
    out.store(dst + hi);
  };

  if (slot >= 0 && slot < a.n_slots) {
    const int pg = (int)a.page.div((unsigned)slot);
    const long long to = pg * a.page_stride + (slot - pg * a.page_size) * a.token_stride;
    for (int t = me; t < nk; t += step) {                   // values: as they are, in the cache's type
      if (t != me) pv = fetch(vrow, t, a.n_kv);
      const int h = t * kHeads + g;
      if (!on || h >= a.n_kv) continue;
      TO* dst = (TO*)a.vc + to + h * a.head_stride;
      if constexpr (sizeof(TI) == sizeof(TO)) {
        pv.lo.store((TI*)(dst + lo));
        pv.hi.store((TI*)(dst + hi));
      } else {
        Run<TO, R> out;
        float x[R];
        pv.lo.get(x); out.put(x); out.store(dst + lo);
        pv.hi.get(x); out.put(x); out.store(dst + hi);
      }
    }
    if (fk < nk) factors(a.k_norm);
    for (int t = fk; t < nk; t += step) {
      if (t != fk) pk = fetch(krow, t, a.n_kv);
      const int h = t * kHeads + g;
      turn(pk, a.k_norm, (TO*)a.kc + to + h * a.head_stride, h < a.n_kv);
    }
  }
  if (fq >= nq) return;
  factors(a.q_norm);
  TO* dst = (TO*)a.q_out + row * a.ldo + (fq * kHeads + g) * hd;
  for (int t = fq; t < nq; t += kDepth * step)
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int u = t + i * step;
      if (u >= nq) return;
      turn(pq[i], a.q_norm, dst, u * kHeads + g < a.n_q);
      dst += step * kHeads * hd;
      if (u + kDepth * step < nq) pq[i] = fetch(qrow, u + kDepth * step, a.n_q);
    }
}

template <typename TI, typename TO>
cudaError_t launch_rope(RopeArgs a, cudaStream_t st) {
  auto go = [&](auto kernel, int lph) {
    // One warp a row from 3552 rows on (24 warps an SM; registers let 16 be
    // resident, so 4096 rows are 1.7 waves), else more, up to one for each group
    // of heads. (A row's table entries and weights cost as much as a few of its
    // heads: with 2 or 4 warps a row, 4096 rows took 26 and 34 us where one a
    // row took 23.)
    const int per = 32 / lph, groups = (a.n_q + per - 1) / per + (a.row_slot ? 2 * ((a.n_kv + per - 1) / per) : 0);
    const long long want = (3551ll + a.rows) / a.rows;
    a.per_row = (int)(want < groups ? want : groups);
    const long long blocks = ((long long)a.rows * a.per_row + kWarps - 1) / kWarps;
    return launch_pdl(kernel, dim3((unsigned)blocks), dim3(kWarps * 32), 0, st, a);
  };
  // runs of 8 where the halves of what rotates and of what does not are whole
  // numbers of them
  if (a.rot % 16 == 0 && (a.hd - a.rot) % 16 == 0) {
    if (a.rot == a.hd) {
      if (a.hd == 64) return go(qk_norm_rope_kernel<TI, TO, 8, 4, true>, 4);
      if (a.hd == 128) return go(qk_norm_rope_kernel<TI, TO, 8, 8, true>, 8);
      if (a.hd == 256) return go(qk_norm_rope_kernel<TI, TO, 8, 16, true>, 16);
    }
    if (a.hd <= 128) return go(qk_norm_rope_kernel<TI, TO, 8, 8, false>, 8);
    return go(qk_norm_rope_kernel<TI, TO, 8, 16, false>, 16);
  }
  if (a.hd <= 64) return go(qk_norm_rope_kernel<TI, TO, 4, 8, false>, 8);
  if (a.hd <= 128) return go(qk_norm_rope_kernel<TI, TO, 4, 16, false>, 16);
  return go(qk_norm_rope_kernel<TI, TO, 4, 32, false>, 32);
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
  if (rot_dim < 0 || rot_dim > hd || rot_dim % 8)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: rot_dim %d (multiples of 8 up to head_dim %d)", who, rot_dim, hd);
  if (rows == 0) return MOE_OK;
  if (n_q && (!q || !q_out)) return at::fail(MOE_ERR_INVALID, "%s: q and q_out are needed", who);
  if (row_slot && (!k || !v)) return at::fail(MOE_ERR_INVALID, "%s: row_slot without k and v", who);
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
  if (n_q == 0 && !row_slot) return MOE_OK;
  // q_out may be q itself; any other overlap would be read after it was written
  const long long nq = (long long)n_q * hd, nk = (long long)cache->n_kv * hd;
  const bool same = q_out == q && ldo == ldq && es == eo;
  if (n_q && !same && at::overlap(q_out, ldo, nq, eo, q, ldq, nq, es, rows))
    return at::fail(MOE_ERR_INVALID, "%s: q_out overlaps q without being q", who);
  if (n_q && row_slot &&
      (at::overlap(q_out, ldo, nq, eo, k, ldk, nk, es, rows) || at::overlap(q_out, ldo, nq, eo, v, ldv, nk, es, rows)))
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
