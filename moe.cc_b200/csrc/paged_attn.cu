// paged_attn.cu — moe_paged_attention_dev: attention of one new token per row
// over a paged key-value cache (the decode form of test_model_trace.c:394-420).
//
//   out_h = sum_t p_t v_t,  p = softmax_t(scale q_h . k_t),  t = 0..position
//
// for every query head h of a row, the key-value head being h / (n_q/n_kv).
//
// Bound: the row's K and V are read once, 2 len n_kv hd elements, and each
// element meets only n_q/n_kv query heads, a few flops per byte: HBM. So the
// kernel is built to keep copies in flight and everything else off the path:
//
//  * One CTA takes a run of positions of one (row, key-value head); all query
//    heads of that key-value head are served by the same reads (up to 8 or 16
//    heads, more take further CTAs that find the run in L2).
//  * Warps are independent: each walks its own 16-position steps through a
//    private ring of cp.async stages (no block barrier in the loop) with its
//    own running maximum and sum; the warps of a CTA are joined once, at the
//    end, and the CTAs of a row by a second, small launch.
//  * Products run on the tensor cores with the operands turned round: the 16
//    positions are the matrix rows of S^T = K Q^T and the query heads its
//    columns, so 8 heads fill an m16n8 tile where Q K^T would pad them to 16.
//    O^T += V^T P^T then has the head dimension as rows. A column of either
//    accumulator is one head and sits in the same lanes, so the softmax
//    rescaling touches no other lane. The m64/m128-row tiles of tcgen05 would
//    be padded 8 to 16 times over here, and the copies bound the kernel anyway.
//  * The running maximum is a reference, not the maximum: it moves only when a
//    score exceeds it by more than 2^8 (one vote per step), since any reference
//    within the exponent's range gives the same softmax.
//
// Precision: scores, maxima, sums and accumulators are fp32. With a 16-bit
// cache the probabilities enter the second product as a sum of two 16-bit
// numbers (a rounding of p and the rounding of its remainder, 2^-17 or better
// together), because one 16-bit p would cost the output as much as its own
// rounding does. With an fp32 cache both products run as three tf32 products
// of high and low parts (the low parts' product, 2^-24, is left out), summed
// from zero per step and added to fp32 sums outside the tensor core.
#include "attn.cuh"

#include <atomic>
#include <type_traits>

namespace moe {
namespace {

constexpr int kMaxParts = 128;      // runs a row is split into at most
constexpr int kMinRun = 64;         // positions of the shortest run
constexpr int kStep = 16;           // positions a warp takes at a time
constexpr float kRaise = 8.0f;      // log2 by which a score may exceed the reference

struct AttnArgs {
  const void *q, *k, *v;
  const int *table, *row_seq, *row_pos;
  void* out;
  float *lse, *part_o;
  float2* part_ml;
  long long ldq, ldo, page_stride, token_stride, head_stride, capacity;
  int rows, n_q, n_kv, group, hd, tiles, n_seq, n_pages, page_size, max_pages, parts;
  float scale_log2;
  at::FastDiv page;
};

// The runs of a row: how many, and how long each (a multiple of 64 so that
// steps never straddle the start of a page that holds a multiple of 16).
struct Runs { int len, run, n; };
__device__ __forceinline__ Runs runs_of(int pos, long long capacity, int parts) {
  Runs r;
  r.len = pos < 0 ? 0 : (int)min((long long)pos + 1, capacity);
  const int even = (r.len + parts - 1) / parts;
  r.run = max(kMinRun, (even + 63) / 64 * 64);
  r.n = r.len ? 1 + (r.len - 1) / r.run : 0;
  return r;
}

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool on) {
  const int n = on ? 16 : 0;        // 0: the 16 bytes are zeroed and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], unsigned p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ unsigned turn8x8(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_tf32(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo with hi a tf32 number (11 bits, nearest) and lo the fp32
// remainder, of which the tensor core reads another 11 bits
__device__ __forceinline__ void split_tf32(float x, unsigned& hi, unsigned& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// (p0, p1) as 16-bit pairs: a rounding and the rounding of its remainder
template <typename T> __device__ __forceinline__ void split16(float p0, float p1, unsigned& hi, unsigned& lo);
template <> __device__ __forceinline__ void split16<__nv_bfloat16>(float p0, float p1, unsigned& hi, unsigned& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
  const __nv_bfloat162 l = __floats2bfloat162_rn(p0 - __low2float(h), p1 - __high2float(h));
  hi = *reinterpret_cast<const unsigned*>(&h);
  lo = *reinterpret_cast<const unsigned*>(&l);
}
template <> __device__ __forceinline__ void split16<__half>(float p0, float p1, unsigned& hi, unsigned& lo) {
  const __half2 h = __floats2half2_rn(p0, p1);
  const __half2 l = __floats2half2_rn(p0 - __low2float(h), p1 - __high2float(h));
  hi = *reinterpret_cast<const unsigned*>(&h);
  lo = *reinterpret_cast<const unsigned*>(&l);
}

template <typename T> __device__ __forceinline__ void store1(void* p, long long i, float v);
template <> __device__ __forceinline__ void store1<float>(void* p, long long i, float v) { ((float*)p)[i] = v; }
template <> __device__ __forceinline__ void store1<__nv_bfloat16>(void* p, long long i, float v) { ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void store1<__half>(void* p, long long i, float v) { ((__half*)p)[i] = __float2half_rn(v); }

// Shapes of one instantiation. HD: head_dim rounded up to 64, 128 or 256 (the
// columns between are zeros in shared memory); NT: 8-head column tiles.
template <typename T, int HD, int NT>
struct Shape {
  static constexpr bool wide = sizeof(T) == 4;
  // Row pitches that make the fragment loads conflict-free: 16-bit rows an odd
  // number of 16-byte pieces (ldmatrix); fp32 K rows 16 words past a multiple
  // of 32 (16-byte loads by 4 lanes of each of 2 rows), V rows 8 words past it
  // (8-byte reach of 4 rows).
  static constexpr int k_pitch = wide ? HD * 4 + 64 : HD * 2 + 16;
  static constexpr int v_pitch = wide ? HD * 4 + 32 : HD * 2 + 16;
  static constexpr int stage = kStep * (k_pitch + v_pitch);
  // 16-bit up to 128: two CTAs of 4 warps on an SM; above, and fp32: one
  static constexpr int warps = wide && HD == 256 ? 2 : 4;
  static constexpr int stages = 3;
  static constexpr int ctas = (wide ? HD <= 64 : HD <= 128) ? 2 : 1;
  static constexpr int heads = 8 * NT;
  static constexpr int q_bytes = wide ? 2 * heads * k_pitch : 0;      // fp32: Q's high and low parts
  static constexpr int ring = warps * stages * stage;
  static constexpr int join = warps * heads * (HD + 2) * 4;
  static constexpr int smem = (ring > join ? ring : join) + q_bytes + 64;
};

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(Shape<T, HD, NT>::warps * 32, Shape<T, HD, NT>::ctas)
paged_attn_kernel(const AttnArgs a) {
  using S = Shape<T, HD, NT>;
  extern __shared__ __align__(16) unsigned char sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  // the small kernel that joins the runs may be scheduled from here on; it
  // waits for this grid's end before it reads
  pdl_launch();

  const int part = blockIdx.x % a.parts;
  int item = blockIdx.x / a.parts;
  const int tile = item % a.tiles; item /= a.tiles;
  const int kvh = item % a.n_kv, row = item / a.n_kv;
  const int seq = a.row_seq ? a.row_seq[row] : row;
  if (seq < 0 || seq >= a.n_seq) return;                       // a padded row: left as it is
  const int head0 = kvh * a.group + tile * S::heads;           // first query head of this CTA
  const int heads = min(S::heads, a.group - tile * S::heads);
  const Runs rn = runs_of(a.row_pos[row], a.capacity, a.parts);
  if (rn.n == 0) {                                             // no position: zeros
    if (part == 0) {
      for (int i = threadIdx.x; i < heads * a.hd; i += S::warps * 32) {
        const int h = i / a.hd;
        store1<T>(a.out, row * a.ldo + (long long)(head0 + h) * a.hd + (i - h * a.hd), 0.f);
      }
      if (a.lse && threadIdx.x < heads) a.lse[(long long)row * a.n_q + head0 + threadIdx.x] = -INFINITY;
    }
    return;
  }
  if (part >= rn.n) return;
  const int t0 = part * rn.run, t1 = min(rn.len, t0 + rn.run);
  const int n_steps = (t1 - t0 + kStep - 1) / kStep;
  const int mine = n_steps > warp ? (n_steps - warp + S::warps - 1) / S::warps : 0;

  unsigned char* ring = sm + warp * (S::stages * S::stage);
  const int* table = a.table + (long long)seq * a.max_pages;
  const T* kbase = (const T*)a.k + kvh * a.head_stride;
  const T* vbase = (const T*)a.v + kvh * a.head_stride;
  constexpr int kPieces = HD * (int)sizeof(T) / 16;            // 16-byte pieces of a row
  const int pieces = a.hd * (int)sizeof(T) / 16;

  // columns from head_dim to HD are zeros throughout: no copy touches them
  if (pieces < kPieces) {
    for (int i = lane; i < S::stages * 2 * kStep * (kPieces - pieces); i += 32) {
      const int c = pieces + i % (kPieces - pieces), r = i / (kPieces - pieces) % kStep;
      const int m = i / (kPieces - pieces) / kStep, st = m >> 1;
      unsigned char* p = ring + st * S::stage + ((m & 1) ? kStep * S::k_pitch + r * S::v_pitch : r * S::k_pitch);
      *reinterpret_cast<uint4*>(p + 16 * c) = make_uint4(0, 0, 0, 0);
    }
  }

  // Page of position `lane & 15` of step i, -1 where there is none; read one
  // step before the copies that need it.
  auto page_at = [&](int i) -> int {
    const int t = t0 + (i * S::warps + warp) * kStep + (lane & 15);
    if (i >= mine || t >= t1) return -1;
    return table[a.page.div((unsigned)t)];
  };
  // valid positions of the stages in flight, two 16-bit masks a word
  unsigned masks[S::stages];
  auto issue = [&](int i, int pg, int st) -> unsigned {
    if (i >= mine) return 0u;
    const int t = t0 + (i * S::warps + warp) * kStep + (lane & 15);
    const bool ok = pg >= 0 && pg < a.n_pages;
    long long off = 0;
    if (ok) off = pg * a.page_stride + (t - (int)a.page.div((unsigned)t) * a.page_size) * a.token_stride;
    const unsigned mask = __ballot_sync(~0u, ok) & 0xffffu;
    const unsigned kd = smem_u32(ring + st * S::stage), vd = kd + kStep * S::k_pitch;
#pragma unroll
    for (int j = 0; j < kStep * kPieces / 32; ++j) {
      const int e = j * 32 + lane, r = e / kPieces, c = e % kPieces;
      const long long o = __shfl_sync(~0u, off, r);
      const bool on = (mask >> r) & 1;
      if (c < pieces) {
        copy16(kd + r * S::k_pitch + 16 * c, (const char*)(kbase + o) + 16 * c, on);
        copy16(vd + r * S::v_pitch + 16 * c, (const char*)(vbase + o) + 16 * c, on);
      }
    }
    return mask;
  };

  // queries: 16-bit as B fragments in registers, fp32 as high and low parts in
  // shared memory (heads beyond the group are zeros)
  unsigned qf[S::wide ? 1 : NT][S::wide ? 1 : HD / 16][2];
  unsigned char* q_sm = sm + (S::ring > S::join ? S::ring : S::join);
  const T* qrow = (const T*)a.q + row * a.ldq + (long long)head0 * a.hd;
  int pg = page_at(0);
#pragma unroll
  for (int i = 0; i < S::stages - 1; ++i) {
    const int next = page_at(i + 1);
    masks[i] = issue(i, pg, i);
    copies_done();
    pg = next;
  }
  masks[S::stages - 1] = 0;
  if constexpr (S::wide) {
    for (int i = threadIdx.x; i < S::heads * HD; i += S::warps * 32) {
      const int h = i / HD, d = i % HD;
      const float x = h < heads && d < a.hd ? ((const float*)qrow)[h * a.hd + d] : 0.f;
      unsigned hi, lo;
      split_tf32(x, hi, lo);
      *reinterpret_cast<unsigned*>(q_sm + h * S::k_pitch + 4 * d) = hi;
      *reinterpret_cast<unsigned*>(q_sm + (S::heads + h) * S::k_pitch + 4 * d) = lo;
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int h = n * 8 + g, d = ks * 16 + 8 * b + 2 * q4;
          qf[n][ks][b] = h < heads && d < a.hd ? *reinterpret_cast<const unsigned*>(qrow + h * a.hd + d) : 0u;
        }
  }
  __syncwarp();

  float o[HD / 16][NT][4];
  float m_ref[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) { m_ref[n][j] = -INFINITY; l[n][j] = 0.f; }
#pragma unroll
    for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[mt][n][j] = 0.f;
  }
  // f16 weights: the reference is set 2^6 low, so that weights of 2^-30 of the
  // largest still round to something
  constexpr float kLift = std::is_same<T, __half>::value ? 6.0f : 0.0f;

  int st = 0, fill = S::stages - 1;
  for (int i = 0; i < mine; ++i) {
    wait_copies<S::stages - 2>();
    __syncwarp();
    // the stage emptied by the step before is filled while this one is used
    {
      const int next = page_at(i + S::stages);
      masks[S::stages - 1] = issue(i + S::stages - 1, pg, fill);
      copies_done();
      pg = next;
    }
    const unsigned mask = masks[0];
    const unsigned char* kst = ring + st * S::stage;
    const unsigned char* vst = kst + kStep * S::k_pitch;

    // S^T: positions g, g+8 (rows) x heads 2 q4, 2 q4 + 1 (columns)
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
    if constexpr (S::wide) {
#pragma unroll 4
      for (int kk = 0; kk < HD / 16; ++kk) {
        // 16 columns: lane q4 holds columns 4 q4 .. 4 q4 + 3, the first two
        // as one k-step of 8, the other two as the next
        const float4 x = *reinterpret_cast<const float4*>(kst + g * S::k_pitch + 64 * kk + 16 * q4);
        const float4 y = *reinterpret_cast<const float4*>(kst + (g + 8) * S::k_pitch + 64 * kk + 16 * q4);
        const uint4 bh = *reinterpret_cast<const uint4*>(q_sm + g * S::k_pitch + 64 * kk + 16 * q4);
        const uint4 bl = *reinterpret_cast<const uint4*>(q_sm + (S::heads + g) * S::k_pitch + 64 * kk + 16 * q4);
        unsigned ah[4], al[4], ch[4], cl[4];
        split_tf32(x.x, ah[0], al[0]); split_tf32(y.x, ah[1], al[1]);
        split_tf32(x.y, ah[2], al[2]); split_tf32(y.y, ah[3], al[3]);
        split_tf32(x.z, ch[0], cl[0]); split_tf32(y.z, ch[1], cl[1]);
        split_tf32(x.w, ch[2], cl[2]); split_tf32(y.w, ch[3], cl[3]);
        float c[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
        mma8_tf32(c, al, bh.x, bh.y);
        mma8_tf32(d, cl, bh.z, bh.w);
        mma8_tf32(c, ah, bl.x, bl.y);
        mma8_tf32(d, ch, bl.z, bl.w);
        mma8_tf32(c, ah, bh.x, bh.y);
        mma8_tf32(d, ch, bh.z, bh.w);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[0][j] += c[j] + d[j];
      }
    } else {
      const unsigned ka = smem_u32(kst) + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::k_pitch + (lane >> 4) * 16;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        unsigned af[4];
        ldsm4(af, ka + ks * 32);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16<T>(s[n], af, qf[n][ks][0], qf[n][ks][1]);
      }
    }
    const bool v0 = (mask >> g) & 1, v1 = (mask >> (g + 8)) & 1;
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = ((j < 2) ? v0 : v1) ? s[n][j] * a.scale_log2 : -INFINITY;
        raise |= s[n][j] > m_ref[n][j & 1] + (kLift + kRaise);
      }
    }
    if (__any_sync(~0u, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(s[n][j], s[n][j + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 16));
          const float to = fmaxf(m_ref[n][j], mx - kLift);
          const float f = m_ref[n][j] == to ? 1.0f : exp2f(m_ref[n][j] - to);   // -inf - -inf is not taken
          m_ref[n][j] = to;
          l[n][j] *= f;
#pragma unroll
          for (int mt = 0; mt < HD / 16; ++mt) { o[mt][n][j] *= f; o[mt][n][j + 2] *= f; }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float m = m_ref[n][j & 1] == -INFINITY ? 0.f : m_ref[n][j & 1];
        s[n][j] = exp2f(s[n][j] - m);
      }
      l[n][0] += s[n][0] + s[n][2];
      l[n][1] += s[n][1] + s[n][3];
    }

    // O^T += V^T P^T
    if constexpr (S::wide) {
      // P^T fragments: position q4 (+4, +8, +12) of head g
      unsigned ph[4], pl[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int src = ((j & 1) * 4 + q4) * 4 + (g >> 1);
        const float e0 = __shfl_sync(~0u, s[0][(j >> 1) * 2], src);
        const float e1 = __shfl_sync(~0u, s[0][(j >> 1) * 2 + 1], src);
        split_tf32((g & 1) ? e1 : e0, ph[j], pl[j]);
      }
#pragma unroll
      for (int b = 0; b < HD / 32; ++b) {
        // 32 columns of V: lane g holds columns 4 g .. 4 g + 3 of the block,
        // the first two as rows g and g + 8 of one tile, the others of the next
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = *reinterpret_cast<const float4*>(vst + (q4 + 4 * j) * S::v_pitch + 128 * b + 16 * g);
        float c[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
        unsigned ah[2][4], al[2][4], ch[2][4], cl[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          split_tf32(x[2 * j].x, ah[j][0], al[j][0]); split_tf32(x[2 * j].y, ah[j][1], al[j][1]);
          split_tf32(x[2 * j + 1].x, ah[j][2], al[j][2]); split_tf32(x[2 * j + 1].y, ah[j][3], al[j][3]);
          split_tf32(x[2 * j].z, ch[j][0], cl[j][0]); split_tf32(x[2 * j].w, ch[j][1], cl[j][1]);
          split_tf32(x[2 * j + 1].z, ch[j][2], cl[j][2]); split_tf32(x[2 * j + 1].w, ch[j][3], cl[j][3]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma8_tf32(c, al[j], ph[2 * j], ph[2 * j + 1]);
          mma8_tf32(d, cl[j], ph[2 * j], ph[2 * j + 1]);
          mma8_tf32(c, ah[j], pl[2 * j], pl[2 * j + 1]);
          mma8_tf32(d, ch[j], pl[2 * j], pl[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma8_tf32(c, ah[j], ph[2 * j], ph[2 * j + 1]);
          mma8_tf32(d, ch[j], ph[2 * j], ph[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[2 * b][0][j] += c[j]; o[2 * b + 1][0][j] += d[j]; }
      }
    } else {
      unsigned ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          unsigned hi, lo;
          split16<T>(s[n][2 * j], s[n][2 * j + 1], hi, lo);
          ph[n][j] = turn8x8(hi);
          pl[n][j] = turn8x8(lo);
        }
      const unsigned va = smem_u32(vst) + ((lane & 7) + (lane >> 4) * 8) * S::v_pitch + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) {
        unsigned af[4];
        ldsm4t(af, va + mt * 32);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16<T>(o[mt][n], af, ph[n][0], ph[n][1]);
          mma16<T>(o[mt][n], af, pl[n][0], pl[n][1]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j + 1 < S::stages; ++j) masks[j] = masks[j + 1];
    st = st + 1 == S::stages ? 0 : st + 1;
    fill = fill + 1 == S::stages ? 0 : fill + 1;
  }

  // ---- join the warps ----
  wait_copies<0>();
  __syncthreads();
  float* jo = reinterpret_cast<float*>(sm);                       // [warp][head][HD]
  float* jm = jo + S::warps * S::heads * HD;                      // [warp][head]
  float* jl = jm + S::warps * S::heads;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float t = l[n][j];
      t += __shfl_xor_sync(~0u, t, 4);
      t += __shfl_xor_sync(~0u, t, 8);
      t += __shfl_xor_sync(~0u, t, 16);
      const int h = n * 8 + 2 * q4 + j;
      if (g == 0) { jm[warp * S::heads + h] = m_ref[n][j]; jl[warp * S::heads + h] = t; }
      float* dst = jo + (warp * S::heads + h) * HD;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int d = S::wide ? (mt >> 1) * 32 + 4 * g + 2 * (mt & 1) + r : mt * 16 + g + 8 * r;
          dst[d] = o[mt][n][j + 2 * r];
        }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (HD / 4); i += S::warps * 32) {
    const int h = i / (HD / 4), d = i % (HD / 4) * 4;
    if (d >= a.hd) continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < S::warps; ++w) m = fmaxf(m, jm[w * S::heads + h]);
    const float m0 = m == -INFINITY ? 0.f : m;
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < S::warps; ++w) {
      const float f = exp2f(jm[w * S::heads + h] - m0);
      const float4 x = *reinterpret_cast<const float4*>(jo + (w * S::heads + h) * HD + d);
      sum = fmaf(f, jl[w * S::heads + h], sum);
      acc[0] = fmaf(f, x.x, acc[0]); acc[1] = fmaf(f, x.y, acc[1]);
      acc[2] = fmaf(f, x.z, acc[2]); acc[3] = fmaf(f, x.w, acc[3]);
    }
    const long long rh = (long long)row * a.n_q + head0 + h;
    if (rn.n == 1) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= inv;
      using V = at::Vec4<T>;
      *reinterpret_cast<typename V::raw*>((T*)a.out + row * a.ldo + (long long)(head0 + h) * a.hd + d) = V::put(acc);
      if (a.lse && d == 0) a.lse[rh] = (m + log2f(sum)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<float4*>(a.part_o + (rh * a.parts + part) * a.hd + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) a.part_ml[rh * a.parts + part] = make_float2(m, sum);
    }
  }
}

// Joins the runs of a row: a block per (row, query head), the runs dealt to
// its 8 warps, each lane four (or eight) elements of the head.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join_kernel(const AttnArgs a) {
  __shared__ float sw[kMaxParts], red[kJoinWarps][256], total;
  const int row = blockIdx.x / a.n_q, h = blockIdx.x % a.n_q;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // every block waits, those without work too: what follows this launch in
  // the stream relies on the first kernel's results being there
  pdl_wait();
  const int seq = a.row_seq ? a.row_seq[row] : row;
  if (seq < 0 || seq >= a.n_seq) return;
  const Runs rn = runs_of(a.row_pos[row], a.capacity, a.parts);
  if (rn.n <= 1) return;
  const long long base = ((long long)row * a.n_q + h) * a.parts;
  if (warp == 0) {
    float2 ml[kMaxParts / 32];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kMaxParts / 32; ++j) {
      const int p = j * 32 + lane;
      ml[j] = p < rn.n ? a.part_ml[base + p] : make_float2(-INFINITY, 0.f);
      m = fmaxf(m, ml[j].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float m0 = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxParts / 32; ++j) {
      const float f = exp2f(ml[j].x - m0);
      sw[j * 32 + lane] = f;
      sum = fmaf(f, ml[j].y, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
      total = sum;
      if (a.lse) a.lse[(long long)row * a.n_q + h] = (m + log2f(sum)) * 0.6931471805599453f;
    }
  }
  __syncthreads();
  for (int d = 4 * lane; d < a.hd; d += 128) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = warp; p < rn.n; p += kJoinWarps) {
      const float f = sw[p];
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + (base + p) * a.hd + d);
      acc[0] = fmaf(f, x.x, acc[0]); acc[1] = fmaf(f, x.y, acc[1]);
      acc[2] = fmaf(f, x.z, acc[2]); acc[3] = fmaf(f, x.w, acc[3]);
    }
    *reinterpret_cast<float4*>(&red[warp][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.hd; d += kJoinWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) x += red[w][d];
    store1<T>(a.out, row * a.ldo + (long long)h * a.hd + d, total == 0.f ? 0.f : x / total);
  }
}

// ---- host side ---------------------------------------------------------------

int head_tile(int dtype, int hd, int group) {
  return dtype != MOE_DTYPE_F32 && hd <= 128 && group > 8 ? 16 : 8;
}

// How many runs a row may be split into. Rows and key-value heads alone that
// fill the GPU's two CTAs per SM need no split for parallelism, but a ragged
// batch does for balance: runs of 512 positions.
int parts_of(int rows, int n_kv, int tiles, int max_kv) {
  const long long items = (long long)rows * n_kv * tiles;
  long long parts = (296 + items - 1) / items;
  if (items >= 4) parts = 296 / items;
  const long long even = (max_kv - 1) / 512 + 1, most = (max_kv - 1) / kMinRun + 1;
  if (rows > 1 && parts < even) parts = even;
  if (parts > most) parts = most;
  if (parts > kMaxParts) parts = kMaxParts;
  return parts < 1 ? 1 : (int)parts;
}

template <typename T, int HD, int NT>
cudaError_t launch_attn(const AttnArgs& a, int device, cudaStream_t st) {
  using S = Shape<T, HD, NT>;
  static std::atomic<unsigned long long> ready{0};       // devices whose limit is raised
  const unsigned long long bit = 1ull << (device & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<T, HD, NT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return e;
    if (device < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  const unsigned grid = (unsigned)((long long)a.rows * a.n_kv * a.tiles * a.parts);
  paged_attn_kernel<T, HD, NT><<<grid, S::warps * 32, S::smem, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || a.parts == 1) return e;
  return launch_pdl(paged_attn_join_kernel<T>, dim3((unsigned)a.rows * (unsigned)a.n_q), dim3(kJoinWarps * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_type(const AttnArgs& a, int tile, int device, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (tile == 16) return a.hd <= 64 ? launch_attn<T, 64, 2>(a, device, st) : launch_attn<T, 128, 2>(a, device, st);
  }
  if (a.hd <= 64) return launch_attn<T, 64, 1>(a, device, st);
  if (a.hd <= 128) return launch_attn<T, 128, 1>(a, device, st);
  return launch_attn<T, 256, 1>(a, device, st);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_paged_attention_workspace(int rows, int n_q, const MoeKvCache* cache, int max_kv) {
  if (at::check_cache(cache, "moe_paged_attention_workspace")) return 0;
  if (rows < 1 || n_q < 1 || n_q % cache->n_kv || max_kv < 1) return 0;
  const int group = n_q / cache->n_kv, ht = head_tile(cache->dtype, cache->head_dim, group);
  const int parts = parts_of(rows, cache->n_kv, (group + ht - 1) / ht, max_kv);
  if (parts == 1) return 0;
  return (size_t)rows * n_q * parts * (sizeof(float2) + sizeof(float) * cache->head_dim) + 16;
}

extern "C" int moe_paged_attention_dev(const void* q, long long ldq, const MoeKvCache* cache, const int* block_table,
                                       int n_seq, int max_pages, const int* row_seq, const int* row_pos, int rows,
                                       int n_q, int max_kv, float scale, void* out, long long ldo, float* lse,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  static const char who[] = "moe_paged_attention_dev";
  int rc = at::check_cache(cache, who);
  if (rc) return rc;
  const int es = at::elem_size(cache->dtype), hd = cache->head_dim;
  if (rows < 0 || n_q < 1 || n_q % cache->n_kv)
    return at::fail(MOE_ERR_INVALID, "%s: rows %d, n_q %d over n_kv %d", who, rows, n_q, cache->n_kv);
  if (n_seq < 0 || max_pages < 1) return at::fail(MOE_ERR_INVALID, "%s: n_seq %d, max_pages %d", who, n_seq, max_pages);
  if (!row_seq && rows > n_seq) return at::fail(MOE_ERR_INVALID, "%s: %d rows of %d sequences need row_seq", who, rows, n_seq);
  if (max_kv < 1) return at::fail(MOE_ERR_INVALID, "%s: max_kv %d", who, max_kv);
  if (rows == 0) return MOE_OK;
  if (!q || !out || !row_pos || !block_table)
    return at::fail(MOE_ERR_INVALID, "%s: q, out, row_pos and block_table are needed", who);
  if (ldq < (long long)n_q * hd || ldo < (long long)n_q * hd)
    return at::fail(MOE_ERR_INVALID, "%s: rows of q or out overlap", who);
  if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || ldq % (16 / es) || ldo % (16 / es))
    return at::fail(MOE_ERR_INVALID, "%s: rows of q and out must start on 16-byte boundaries", who);
  const int group = n_q / cache->n_kv, ht = head_tile(cache->dtype, hd, group);
  AttnArgs a{};
  a.tiles = (group + ht - 1) / ht;
  a.parts = parts_of(rows, cache->n_kv, a.tiles, max_kv);
  if ((long long)rows * cache->n_kv * a.tiles * a.parts > INT32_MAX || (long long)rows * n_q > INT32_MAX)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: too many rows and heads for one launch", who);
  const size_t need = moe_paged_attention_workspace(rows, n_q, cache, max_kv);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return at::fail(MOE_ERR_INVALID, "%s: %zu bytes of 16-byte aligned workspace are needed, %zu given", who, need,
                    workspace ? workspace_bytes : (size_t)0);
  at::OnDeviceOf on;
  if ((rc = on.enter(q, who))) return rc;
  a.q = q; a.k = cache->k; a.v = cache->v; a.table = block_table; a.row_seq = row_seq; a.row_pos = row_pos;
  a.out = out; a.lse = lse; a.ldq = ldq; a.ldo = ldo;
  a.page_stride = cache->page_stride; a.token_stride = cache->token_stride; a.head_stride = cache->head_stride;
  a.capacity = (long long)max_pages * cache->page_size;
  if (a.capacity > INT32_MAX - 1024) a.capacity = INT32_MAX - 1024;   // positions stay ints through a run's end
  a.rows = rows; a.n_q = n_q; a.n_kv = cache->n_kv; a.group = group; a.hd = hd; a.n_seq = n_seq;
  a.n_pages = cache->n_pages; a.page_size = cache->page_size; a.max_pages = max_pages;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.page = at::FastDiv((unsigned)cache->page_size);
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)((char*)workspace + ((size_t)rows * n_q * a.parts * hd * sizeof(float) + 15) / 16 * 16);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (cache->dtype == MOE_DTYPE_BF16) e = launch_type<__nv_bfloat16>(a, ht, on.device(), st);
  else if (cache->dtype == MOE_DTYPE_F16) e = launch_type<__half>(a, ht, on.device(), st);
  else e = launch_type<float>(a, ht, on.device(), st);
  if (e != cudaSuccess) { cudaGetLastError(); return at::fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e)); }
  return MOE_OK;
}
