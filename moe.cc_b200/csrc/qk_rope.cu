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
// The bound is bytes: every element is read once and written once. A head is
// held by LPH lanes, each with four elements of the lower half and the four
// that rotate with them from the upper half, so the rotation needs no
// exchange between lanes and the mean is a shuffle sum. A block takes one row:
// its lanes load the weights and the row's table entries once and then walk
// over the row's heads.
#include "attn.cuh"

namespace moe {
namespace {

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *kc, *vc;
  const float *q_norm, *k_norm, *rope;
  const int *row_pos, *row_slot;
  long long ldq, ldk, ldv, ldo, page_stride, token_stride, head_stride;
  int n_q, n_kv, hd, rot, rope_len, n_slots, page_size;
  float eps;
  at::FastDiv page;
};

constexpr int kThreads = 128;

template <typename TI, typename TO, int LPH>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch();
  using VI = at::Vec4<TI>;
  using VO = at::Vec4<TO>;
  const int row = blockIdx.x, g = threadIdx.x / LPH, l = threadIdx.x % LPH;
  const int pos = a.row_pos ? a.row_pos[row] : 0;
  if (pos < 0 || (a.rot && pos >= a.rope_len)) return;      // a padded row: nothing of it is touched
  const bool on = 4 * l < a.hd / 2;
  // this lane's four pairs (lo + t, hi + t)
  int lo = 4 * l, hi = 4 * l + a.rot / 2;
  const bool turns = lo < a.rot / 2;
  if (!turns) { lo = 4 * l + a.rot / 2; hi = lo + (a.hd - a.rot) / 2; }
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (on && turns) {
    const float* t = a.rope + (long long)pos * a.rot + lo;
    at::Vec4<float>::get(*reinterpret_cast<const float4*>(t), c);
    at::Vec4<float>::get(*reinterpret_cast<const float4*>(t + a.rot / 2), s);
  }
  long long at_slot = -1;
  if (a.row_slot) {
    const int slot = a.row_slot[row];
    if (slot >= 0 && slot < a.n_slots) {
      const int pg = (int)a.page.div((unsigned)slot);
      at_slot = pg * a.page_stride + (slot - pg * a.page_size) * a.token_stride;
    }
  }
  const int heads = a.n_q + (at_slot >= 0 ? 2 * a.n_kv : 0);   // without a slot only the queries are worked on
  const int step = gridDim.y * (kThreads / LPH);
  int h = blockIdx.y * (kThreads / LPH) + g;
  // the loop runs alike for all groups of a warp (the sum below shuffles)
  for (int base = blockIdx.y * (kThreads / LPH); base < heads; base += step, h += step) {
    const bool live = on && h < heads;
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
    const int kvh = is_k ? h - a.n_q : h - a.n_q - a.n_kv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
      const TI* src = is_q ? (const TI*)a.q + row * a.ldq + (long long)h * a.hd
                    : is_k ? (const TI*)a.k + row * a.ldk + (long long)kvh * a.hd
                           : (const TI*)a.v + row * a.ldv + (long long)kvh * a.hd;
      VI::get(*reinterpret_cast<const typename VI::raw*>(src + lo), x);
      VI::get(*reinterpret_cast<const typename VI::raw*>(src + hi), x + 4);
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
    if (!live) continue;
    const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    if (w) {
      const float inv = 1.0f / sqrtf(sq / (float)a.hd + a.eps);
      float wl[8];
      at::Vec4<float>::get(*reinterpret_cast<const float4*>(w + lo), wl);
      at::Vec4<float>::get(*reinterpret_cast<const float4*>(w + hi), wl + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wl[i];
    }
    if (is_q || is_k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = x[i], o = x[i + 4];
        if (turns) {
          x[i] = e * c[i] - o * s[i];
          x[i + 4] = o * c[i] + e * s[i];
        }
      }
    }
    TO* dst = is_q ? (TO*)a.q_out + row * a.ldo + (long long)h * a.hd
                   : (is_k ? (TO*)a.kc : (TO*)a.vc) + at_slot + kvh * a.head_stride;
    *reinterpret_cast<typename VO::raw*>(dst + lo) = VO::put(x);
    *reinterpret_cast<typename VO::raw*>(dst + hi) = VO::put(x + 4);
  }
}

template <typename TI, typename TO>
cudaError_t launch_rope(const RopeArgs& a, int rows, cudaStream_t st) {
  const int heads = a.n_q + 2 * a.n_kv;
  auto go = [&](auto kernel, int lph) {
    // few rows: one head per lane group, so that the row spreads over blocks;
    // many rows: a block keeps its row's table entries for all heads
    const int per = kThreads / lph, full = (heads + per - 1) / per;
    const int y = rows >= 1184 ? 1 : full;
    return launch_pdl(kernel, dim3(rows, y), dim3(kThreads), 0, st, a);
  };
  if (a.hd <= 64) return go(qk_norm_rope_kernel<TI, TO, 8>, 8);
  if (a.hd <= 128) return go(qk_norm_rope_kernel<TI, TO, 16>, 16);
  return go(qk_norm_rope_kernel<TI, TO, 32>, 32);
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
  a.n_q = n_q; a.n_kv = cache->n_kv; a.hd = hd; a.rot = rot_dim; a.rope_len = rope_len;
  a.n_slots = cache->n_pages * cache->page_size; a.page_size = cache->page_size; a.eps = eps;
  a.page = at::FastDiv((unsigned)cache->page_size);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == MOE_DTYPE_BF16) e = launch_rope<__nv_bfloat16, __nv_bfloat16>(a, rows, st);
  else if (dtype == MOE_DTYPE_F16) e = launch_rope<__half, __half>(a, rows, st);
  else if (cache->dtype == MOE_DTYPE_F32) e = launch_rope<float, float>(a, rows, st);
  else if (cache->dtype == MOE_DTYPE_BF16) e = launch_rope<float, __nv_bfloat16>(a, rows, st);
  else e = launch_rope<float, __half>(a, rows, st);
  return at::launched(e, who);
}
