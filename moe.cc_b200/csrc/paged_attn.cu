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
// of high and low parts (the low parts' product, 2^-24, is left out). Products
// are summed from zero per step and added to fp32 sums outside the tensor core,
// whose sums truncate: kept inside over 2048 steps they took 2.3e-4 off values
// of one sign, as much as an f16 rounding (now 6e-7; the additions cost 0 to
// 1.5 % of the time).
//
// An operand in two parts is not what it was where it is infinite (inf - inf is
// no remainder, and inf times a remainder of 0 is NaN). A warp whose sums come
// out NaN therefore takes its run again with plain fp32 products (attend, "NaN").
#include "attn.cuh"

#include <float.h>

#include <atomic>
#include <type_traits>

namespace moe {
namespace {

constexpr int kMaxParts = 128;      // runs a row is split into at most
constexpr int kPiece = 64;          // positions of the shortest run
constexpr int kDealtRows = 512;     // rows whose work is dealt evenly
constexpr int kRun = 8;             // pieces of the shortest run of more rows
constexpr int kRowParts = 16384;    // parts of all of them together
constexpr int kShort = 32;          // pieces up to which a cluster takes a row
constexpr int kCluster = 8;         // CTAs of such a cluster at most
enum { kRuns = 0, kDealt = 1, kClustered = 2 };
constexpr int kStep = 16;           // positions a warp takes at a time
constexpr float kRaise = 8.0f;      // log2 by which a score may exceed the reference

struct AttnArgs {
  const void *q, *k, *v;
  const int *table, *row_seq, *row_pos;
  void* out;
  float *lse, *part_o;
  float2* part_ml;
  long long ldq, ldo, page_stride, token_stride, head_stride, capacity;
  int rows, n_q, n_kv, group, hd, tiles, n_seq, n_pages, page_size, max_pages;
  int parts;          // partial results that a row's head has room for
  int mode;           // how the work is split (paged_attn_kernel)
  float scale_log2;
  at::FastDiv page;
};

// Positions are dealt out in pieces of 64 (steps of 16 then never straddle the
// start of a page that holds a multiple of 16).
__device__ __forceinline__ int length_of(const AttnArgs& a, int row) {
  const int seq = a.row_seq ? a.row_seq[row] : row;
  if (seq < 0 || seq >= a.n_seq) return -1;                    // a padded row: left as it is
  const int pos = a.row_pos[row];
  return pos < 0 ? 0 : (int)min((long long)pos + 1, a.capacity);
}
__device__ __forceinline__ int pieces_of(int len) { return len > 0 ? (len - 1) / kPiece + 1 : 0; }

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool on) {
  const int n = on ? 16 : 0;        // 0: the 16 bytes are zeroed and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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

// x = hi + lo with hi the nearest number of 11 bits, which is what tf32 holds,
// and lo the exact rest, of which the tensor core reads another 11 bits. (Cut
// off instead of rounded, hi leaves a rest of x's own sign, and what the tensor
// core drops of it adds up: 1.2e-6 instead of 4 to 5e-7 of the output.) From
// 2^128 (1 - 2^-12) on hi is infinite and lo NaN or infinite.
__device__ __forceinline__ void split_tf32(float x, unsigned& hi, unsigned& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
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

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float value(const __half* p) { return __half2float(*p); }

template <typename T> __device__ __forceinline__ void store1(void* p, long long i, float v);
template <> __device__ __forceinline__ void store1<float>(void* p, long long i, float v) { ((float*)p)[i] = v; }
template <> __device__ __forceinline__ void store1<__nv_bfloat16>(void* p, long long i, float v) { ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void store1<__half>(void* p, long long i, float v) { ((__half*)p)[i] = __float2half_rn(v); }

// Shapes of one instantiation. HD: head_dim rounded up to 64, 96, 128 or 256 (the
// columns between are zeros in shared memory); NT: 8-head column tiles.
template <typename T, int HD, int NT>
struct Shape {
  static constexpr bool wide = sizeof(T) == 4;
  // Piece c (16 bytes) of row r lies at c ^ turn(r) of the row, so that the
  // fragment loads meet no bank conflicts: 16-bit rows are read 8 at a time at
  // one piece (ldmatrix), fp32 rows 4 pieces of 2 rows (K: rows two apart, see
  // swap01) or 2 pieces of 4 rows (V) at a time. Rows pitched by an odd number
  // of pieces would do too, but then every other row's 32-byte sectors are
  // not aligned blocks and cross the crossbar twice.
  static constexpr int pitch = HD * (int)sizeof(T);
  static __device__ __forceinline__ constexpr int turn(int r) {
    return wide ? 2 * (r & 3) : HD == 96 ? (r >> 1) & 3 : r & 7;   // 96: rows alternate between the banks' halves
  }
  static constexpr int unit = kStep * pitch;       // the K or the V rows of a step
  // Warps, ring units a warp and CTAs an SM: 8 to 16 warps. 16-bit rows of
  // 128, 32 rows of up to 8192 positions / one row of 131072: 3 CTAs of 4 warps
  // 59.4 / 49.1 us, 2 of 4 60.8 / 49.0, 4 of 4 60.2 / 48.7, 1 of 8 64.5 / 50.0, 5
  // units in 2 CTAs of 4 60.7 / 49.5. fp32, 32 rows of 2048 positions (268 MB):
  // rows of 64 in 1 CTA of 8 warps with 5 units 97 us, 4 of 4 with 3 54; of 128
  // in 2 of 4 with 3 73, 3 of 4 with 2 66; of 256 in 1 of 4 with 3 119, of 6 with
  // 2 104.
  static constexpr int warps = HD == 256 ? wide ? 6 : 8 : 4;
  static constexpr int units = wide ? HD == 64 ? 3 : 2 : HD == 64 || NT == 2 ? 5 : 3;
  static constexpr int ctas = HD == 256 ? 1 : wide ? HD == 64 ? 4 : 3 : NT == 2 ? 2 : HD == 96 ? 4 : 3;
  static constexpr int heads = 8 * NT;
  static constexpr int q_pitch = HD * 4 + 64;      // fp32: Q's high and low parts (4 pieces of 2 rows a load)
  static constexpr int q_bytes = wide ? 2 * heads * q_pitch : 0;
  static constexpr int ring = warps * units * unit;
  static constexpr int join = warps * heads * (HD + 2) * 4;
  static constexpr int both = join + heads * (HD + 2) * 4;   // and the CTA's own result, for its cluster
  static constexpr int base = ring > both ? ring : both;
  static constexpr int smem = base + q_bytes;
};

// K row (position within the step) that matrix row g of the fp32 path holds:
// g with its two lowest bits exchanged, so that the rows of one 16-byte load
// phase lie two pitches apart
__device__ __forceinline__ int swap01(int g) { return (g & 4) | ((g & 1) << 1) | ((g >> 1) & 1); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// what CTA `rank` of the cluster has at p in its shared memory
__device__ __forceinline__ unsigned remote(const float* p, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 remote2(const float* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 remote4(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote(p, rank)) : "memory");
  return v;
}

// Four elements of a row's result, and its lse with the first.
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int row, int head, int d, float (&acc)[4], float sum, float m) {
  using V = at::Vec4<T>;
  const float inv = 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = sum == 0.f ? 0.f : acc[e] * inv;
  *reinterpret_cast<typename V::raw*>((T*)a.out + row * a.ldo + (long long)head * a.hd + d) = V::put(acc);
  if (a.lse && d == 0) a.lse[(long long)row * a.n_q + head] = (m + log2f(sum)) * 0.6931471805599453f;
}

// One run: positions [t0, t1) of one row for one tile of one key-value head's
// query heads, `part` of `parts` such runs.
template <typename T, int HD, int NT>
__device__ __forceinline__ void attend(const AttnArgs& a, unsigned char* sm, int row, int kvh, int tile, int t0, int t1,
                                       int part, int parts) {
  using S = Shape<T, HD, NT>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  const int seq = a.row_seq ? a.row_seq[row] : row;
  const int head0 = kvh * a.group + tile * S::heads;           // first query head
  const int heads = min(S::heads, a.group - tile * S::heads);
  const int n_steps = (t1 - t0 + kStep - 1) / kStep;
  const int mine = n_steps > warp ? (n_steps - warp + S::warps - 1) / S::warps : 0;

  unsigned char* ring = sm + warp * (S::units * S::unit);
  const int* table = a.table + (long long)seq * a.max_pages;
  constexpr int kRow = HD * (int)sizeof(T) / 16;               // 16-byte pieces of a row
  constexpr int kPieces = kRow == 12 ? 16 : kRow == 24 ? 32 : kRow;   // and the lanes that copy one
  const int pieces = a.hd * (int)sizeof(T) / 16;
  const char* kbase = (const char*)((const T*)a.k + kvh * a.head_stride);
  const char* vbase = (const char*)((const T*)a.v + kvh * a.head_stride);
  const long long row_bytes = a.token_stride * (long long)sizeof(T);
  const bool whole = a.page_size % kStep == 0;                 // a step never leaves its page

  // columns from head_dim to HD are zeros throughout: no copy touches them
  if (pieces < kRow) {
    const int pad = kRow - pieces;
    for (int i = lane; i < S::units * kStep * pad; i += 32) {
      const int r = i / pad, c = pieces + i % pad;
      *reinterpret_cast<uint4*>(ring + r * S::pitch + 16 * (c ^ S::turn(r))) = make_uint4(0, 0, 0, 0);
    }
  }

  // Page of step i (of position `lane & 15` of it, where a step may span
  // pages), -1 where there is none. Read one step before the copies need it.
  auto page_at = [&](int i) -> int {
    const int t = t0 + (i * S::warps + warp) * kStep + (whole ? 0 : (lane & 15));
    if (i >= mine || t >= t1) return -1;
    return table[a.page.div((unsigned)t)];
  };
  // Copies the K or V rows of step i to a unit of the ring and returns the mask
  // of the step's positions that are attended; the others' rows become zeros.
  constexpr int kRows = kPieces <= 32 ? 32 / kPieces : 1;      // rows one instruction of the warp covers
  constexpr int kInsn = kStep * kPieces / 32;
  const int r0 = kPieces <= 32 ? lane / kPieces : 0, c0 = kPieces <= 32 ? lane % kPieces : lane;
  const int d0 = r0 * S::pitch + 16 * (c0 ^ S::turn(r0));
  // where this lane's piece of row r0 + r goes (kRows is a power of two and
  // r0 < kRows, so turn(r0 + r) is turn(r0) ^ turn(r))
  auto place = [&](int r, int c) { return (d0 ^ (16 * S::turn(r))) + r * S::pitch + 16 * c; };
  auto issue = [&](const char* base, int i, int pg, int slot) -> unsigned {
    if (i >= mine) return 0u;
    const int t = t0 + (i * S::warps + warp) * kStep;
    const bool ok = pg >= 0 && pg < a.n_pages;
    const unsigned to = smem_u32(ring + slot * S::unit);
    if (whole) {
      const int n = ok ? min(kStep, t1 - t) : 0;
      const int in = t - (int)a.page.div((unsigned)t) * a.page_size;
      const char* src = base + (ok ? pg * a.page_stride * (long long)sizeof(T) + (in + r0) * row_bytes : 0) + 16 * c0;
      if (n == kStep && (kPieces <= 32 || pieces == kPieces)) {   // the usual step: nothing to mask
        if (c0 < pieces) {
#pragma unroll
          for (int j = 0; j < kInsn; ++j) {
            const int r = kPieces <= 32 ? j * kRows : j / 2, c = kPieces <= 32 ? 0 : 32 * (j & 1);
            copy16(to + place(r, c), src + 16 * c);
            if (kPieces <= 32 || (j & 1)) src += kRows * row_bytes;
          }
        }
        return 0xffffu;
      }
#pragma unroll 1
      for (int j = 0; j < kInsn; ++j) {
        const int r = kPieces <= 32 ? j * kRows : j / 2, c = kPieces <= 32 ? 0 : 32 * (j & 1);
        if (c0 + c < pieces) copy16(to + place(r, c), src + r * row_bytes + 16 * c, r0 + r < n);
      }
      return (1u << n) - 1u;
    }
    const int tl = t + (lane & 15);
    long long off = 0;
    if (ok) off = pg * a.page_stride * (long long)sizeof(T) + (tl - (int)a.page.div((unsigned)tl) * a.page_size) * row_bytes;
    const unsigned mask = __ballot_sync(~0u, ok) & 0xffffu;
#pragma unroll
    for (int j = 0; j < kInsn; ++j) {
      const int r = kPieces <= 32 ? j * kRows : j / 2, c = kPieces <= 32 ? 0 : 32 * (j & 1);
      const long long o = __shfl_sync(~0u, off, r0 + r);
      if (c0 + c < pieces) copy16(to + place(r, c), base + o + 16 * (c0 + c), (mask >> (r0 + r)) & 1);
    }
    return mask;
  };

  // The ring holds units K0 V0 K1 V1 ..., kAhead of them in flight; unit u lies
  // in slot u % units, and the copy of unit u + kAhead goes into the slot that
  // unit u - 1 has just left. For an even kAhead, K and V of step i are followed
  // by K and V of step i + kSteps; for an odd one K by V and V by the next K.
  constexpr int kAhead = S::units - 1, kSteps = kAhead / 2;
  constexpr bool kOdd = kAhead & 1;
  unsigned masks[kSteps + 1];                                  // of steps i, i + 1, ...
  int pg = page_at(0);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int next = page_at(i + 1);
    masks[i] = issue(kbase, i, pg, 2 * i);
    copies_done();
    issue(vbase, i, pg, 2 * i + 1);
    copies_done();
    pg = next;
  }
  if constexpr (kOdd) {
    masks[kSteps] = issue(kbase, kSteps, pg, 2 * kSteps);
    copies_done();
  }

  // queries: 16-bit as B fragments in registers, fp32 as high and low parts in
  // shared memory (heads beyond the group are zeros)
  unsigned qf[S::wide ? 1 : NT][S::wide ? 1 : HD / 16][2];
  unsigned char* q_sm = sm + S::base;
  const T* qrow = (const T*)a.q + row * a.ldq + (long long)head0 * a.hd;
  if constexpr (S::wide) {
    for (int i = threadIdx.x; i < S::heads * HD; i += S::warps * 32) {
      const int h = i / HD, d = i % HD;
      const float x = h < heads && d < a.hd ? ((const float*)qrow)[h * a.hd + d] : 0.f;
      unsigned hi, lo;
      split_tf32(x, hi, lo);
      *reinterpret_cast<unsigned*>(q_sm + h * S::q_pitch + 4 * d) = hi;
      *reinterpret_cast<unsigned*>(q_sm + (S::heads + h) * S::q_pitch + 4 * d) = lo;
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

  // Per head (columns 2 q4 + j of tile n): the reference m, which starts below
  // every score, the sum l of this lane's weights, the accumulators.
  float o[HD / 16][NT][4];
  float m_ref[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) { m_ref[n][j] = -FLT_MAX; l[n][j] = 0.f; }
#pragma unroll
    for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[mt][n][j] = 0.f;
  }
  // f16 weights: the reference is set 2^6 low, so that weights of 2^-30 of the
  // largest still round to something
  constexpr float kLift = std::is_same<T, __half>::value ? 6.0f : 0.0f;

  int slot = 0;
  auto before = [&](int s) { return s == 0 ? S::units - 1 : s - 1; };
  auto after = [&](int s) { return s + 1 == S::units ? 0 : s + 1; };
  for (int i = 0; i < mine; ++i) {
    wait_copies<kAhead - 1>();
    __syncwarp();
    const int next = page_at(i + kSteps + 1);
    if constexpr (kOdd) issue(vbase, i + kSteps, pg, before(slot));
    else masks[kSteps] = issue(kbase, i + kSteps, pg, before(slot));
    copies_done();
    const unsigned mask = masks[0];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) masks[j] = masks[j + 1];
    const unsigned char* kst = ring + slot * S::unit;
    slot = after(slot);

    // S^T: positions g, g + 8 (rows) x heads 2 q4, 2 q4 + 1 (columns)
    float s[NT][4];
    if constexpr (S::wide) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0][j] = 0.f;
#pragma unroll 4
      for (int kk = 0; kk < HD / 16; ++kk) {
        // 16 columns: lane q4 holds columns 4 q4 .. 4 q4 + 3, the first two
        // as one k-step of 8, the other two as the next
        const unsigned char* at = kst + swap01(g) * S::pitch + ((64 * kk + 16 * q4) ^ (16 * S::turn(swap01(g))));
        const float4 x = *reinterpret_cast<const float4*>(at);
        const float4 y = *reinterpret_cast<const float4*>(at + 8 * S::pitch);
        const uint4 bh = *reinterpret_cast<const uint4*>(q_sm + g * S::q_pitch + 64 * kk + 16 * q4);
        const uint4 bl = *reinterpret_cast<const uint4*>(q_sm + (S::heads + g) * S::q_pitch + 64 * kk + 16 * q4);
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
      // two accumulators a tile: half the chain of dependent products
      const unsigned ka = smem_u32(kst) + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::pitch;
      const unsigned kx = 16 * ((lane >> 4) ^ S::turn(lane));
      float e[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = e[n][j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ks += 2) {
        unsigned af[4], bf[4];
        ldsm4(af, ka + (kx ^ (ks * 32)));
        ldsm4(bf, ka + (kx ^ (ks * 32 + 32)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16<T>(s[n], af, qf[n][ks][0], qf[n][ks][1]);
          mma16<T>(e[n], bf, qf[n][ks + 1][0], qf[n][ks + 1][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] += e[n][j];
    }
    if (mask != 0xffffu) {
      const int gt = S::wide ? swap01(g) : g;
      const bool v0 = (mask >> gt) & 1, v1 = (mask >> (gt + 8)) & 1;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = ((j < 2) ? v0 : v1) ? s[n][j] * a.scale_log2 : -INFINITY;
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] *= a.scale_log2;
    }
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) raise |= fmaxf(s[n][j], s[n][j + 2]) - m_ref[n][j] > kLift + kRaise;
    if (__any_sync(~0u, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(s[n][j], s[n][j + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 16));
          const float to = fmaxf(m_ref[n][j], mx - kLift), f = ex2(m_ref[n][j] - to);
          m_ref[n][j] = to;
          l[n][j] *= f;
#pragma unroll
          for (int mt = 0; mt < HD / 16; ++mt) { o[mt][n][j] *= f; o[mt][n][j + 2] *= f; }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = ex2(s[n][j] - m_ref[n][j & 1]);
      l[n][0] += s[n][0] + s[n][2];
      l[n][1] += s[n][1] + s[n][3];
    }

    wait_copies<kAhead - 1>();
    __syncwarp();
    if constexpr (kOdd) masks[kSteps] = issue(kbase, i + kSteps + 1, next, before(slot));
    else issue(vbase, i + kSteps, pg, before(slot));
    copies_done();
    pg = next;
    const unsigned char* vst = ring + slot * S::unit;
    slot = after(slot);
    // O^T += V^T P^T
    if constexpr (S::wide) {
      // P^T fragments: position q4 (+4, +8, +12) of head g
      unsigned ph[4], pl[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int src = swap01((j & 1) * 4 + q4) * 4 + (g >> 1);
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
          x[j] = *reinterpret_cast<const float4*>(vst + (q4 + 4 * j) * S::pitch + ((128 * b + 16 * g) ^ (16 * S::turn(q4))));
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
      const unsigned va = smem_u32(vst) + ((lane & 7) + (lane >> 4) * 8) * S::pitch;
      const unsigned vx = 16 * (((lane >> 3) & 1) ^ S::turn(lane));
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) {
        unsigned af[4];
        ldsm4t(af, va + (vx ^ (mt * 32)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          mma16<T>(c, af, pl[n][0], pl[n][1]);
          mma16<T>(c, af, ph[n][0], ph[n][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[mt][n][j] += c[j];
        }
      }
    }
  }

  // ---- join the warps ----
  wait_copies<0>();
  __syncthreads();
  float* jo = reinterpret_cast<float*>(sm);                       // [warp][head][HD]
  float* jm = jo + S::warps * S::heads * HD;                      // [warp][head]
  float* jl = jm + S::warps * S::heads;
  float *co = jl + S::warps * S::heads, *cm = co + S::heads * HD;   // clustered: the CTA's result
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
  // NaN: the warp's steps again, position by position, a head after another.
  // Nothing of a head's sums has to be found infinite for it: an infinite value
  // that met only positive parts is infinite already.
  bool nan = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float t = 0.f;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) t += o[mt][n][j] + o[mt][n][j + 2];
      nan |= n * 8 + 2 * q4 + j < heads && t != t;
    }
  if (__any_sync(~0u, nan)) {
    __syncwarp();
    constexpr int kD = HD / 32;                                   // elements of a head in a lane
#pragma unroll 1
    for (int h = 0; h < heads; ++h) {
      float x[kD], acc[kD], m = -FLT_MAX, sum = 0.f;
#pragma unroll
      for (int e = 0; e < kD; ++e) {
        const int d = lane + 32 * e;
        x[e] = d < a.hd ? value(qrow + h * a.hd + d) : 0.f;
        acc[e] = 0.f;
      }
#pragma unroll 1
      for (int i = 0; i < mine * kStep; ++i) {
        const int t = t0 + (i / kStep * S::warps + warp) * kStep + i % kStep;
        if (t >= t1) break;                                       // the last step's end
        const int pi = (int)a.page.div((unsigned)t), page = table[pi];
        if (page < 0 || page >= a.n_pages) continue;
        const long long at = page * a.page_stride + (t - pi * a.page_size) * a.token_stride;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < kD; ++e)
          if (lane + 32 * e < a.hd) s = fmaf(x[e], value((const T*)kbase + at + lane + 32 * e), s);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
        s *= a.scale_log2;
        if (s > m) {
          const float f = ex2(m - s);
          m = s;
          sum *= f;
#pragma unroll
          for (int e = 0; e < kD; ++e) acc[e] *= f;
        }
        const float p = ex2(s - m);
        sum += p;
#pragma unroll
        for (int e = 0; e < kD; ++e)
          if (lane + 32 * e < a.hd) acc[e] = fmaf(p, value((const T*)vbase + at + lane + 32 * e), acc[e]);
      }
      if (lane == 0) { jm[warp * S::heads + h] = m; jl[warp * S::heads + h] = sum; }
#pragma unroll
      for (int e = 0; e < kD; ++e) jo[(warp * S::heads + h) * HD + lane + 32 * e] = acc[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (HD / 4); i += S::warps * 32) {
    const int h = i / (HD / 4), d = i % (HD / 4) * 4;
    if (d >= a.hd) continue;
    float m = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < S::warps; ++w) m = fmaxf(m, jm[w * S::heads + h]);
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < S::warps; ++w) {
      const float f = ex2(jm[w * S::heads + h] - m);
      const float4 x = *reinterpret_cast<const float4*>(jo + (w * S::heads + h) * HD + d);
      sum = fmaf(f, jl[w * S::heads + h], sum);
      acc[0] = fmaf(f, x.x, acc[0]); acc[1] = fmaf(f, x.y, acc[1]);
      acc[2] = fmaf(f, x.z, acc[2]); acc[3] = fmaf(f, x.w, acc[3]);
    }
    const long long rh = (long long)row * a.n_q + head0 + h;
    if (parts == 1) {
      store_out<T>(a, row, head0 + h, d, acc, sum, m);
      if (d == 0 && a.mode != kClustered && a.parts > 1) a.part_ml[rh * a.parts] = make_float2(m, -0.f);
    } else if (a.mode == kClustered) {
      *reinterpret_cast<float4*>(co + h * HD + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) { cm[2 * h] = m; cm[2 * h + 1] = sum; }
    } else {
      *reinterpret_cast<float4*>(a.part_o + (rh * a.parts + part) * a.hd + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      // the sign of l marks a row's last run (the sum itself is not negative)
      const unsigned mark = part == parts - 1 ? 1u << 31 : 0u;
      if (d == 0)
        a.part_ml[rh * a.parts + part] = make_float2(m, __uint_as_float((__float_as_uint(sum) & 0x7fffffffu) | mark));
    }
  }
  if (a.mode != kClustered || parts == 1) return;
  // ---- join the cluster's CTAs, each of them a share of the elements ----
  cluster_sync();
  for (int i = part * S::warps * 32 + threadIdx.x; i < heads * (HD / 4); i += parts * S::warps * 32) {
    const int h = i / (HD / 4), d = i % (HD / 4) * 4;
    if (d >= a.hd) continue;
    float2 ml[kCluster];
    float4 x[kCluster];
    float m = -FLT_MAX;
#pragma unroll
    for (int p = 0; p < kCluster; ++p) {
      ml[p] = p < parts ? remote2(cm + 2 * h, p) : make_float2(-FLT_MAX, 0.f);
      x[p] = p < parts ? remote4(co + h * HD + d, p) : make_float4(0.f, 0.f, 0.f, 0.f);
      m = fmaxf(m, ml[p].x);
    }
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < kCluster; ++p) {
      const float f = ex2(ml[p].x - m);
      sum = fmaf(f, ml[p].y, sum);
      acc[0] = fmaf(f, x[p].x, acc[0]); acc[1] = fmaf(f, x[p].y, acc[1]);
      acc[2] = fmaf(f, x[p].z, acc[2]); acc[3] = fmaf(f, x[p].w, acc[3]);
    }
    store_out<T>(a, row, head0 + h, d, acc, sum, m);
  }
}

// A row without positions: zeros.
template <typename T>
__device__ __forceinline__ void clear_heads(const AttnArgs& a, int row, int head0, int heads) {
  for (int i = threadIdx.x; i < heads * a.hd; i += blockDim.x)
    store1<T>(a.out, row * a.ldo + (long long)head0 * a.hd + i, 0.f);
  if (a.lse)
    for (int h = threadIdx.x; h < heads; h += blockDim.x) a.lse[(long long)row * a.n_q + head0 + h] = -INFINITY;
}

// How the work is split, an "item" being a row's key-value head and tile:
//   kDealt      The CTAs are taken in groups, one for each key-value head (and
//               tile), and the pieces of all rows, one row after another, are
//               cut into as many stretches, equal to a piece, as there are
//               groups, which is what the GPU holds at a time. A stretch may end
//               one row and begin the next, so a ragged batch leaves no CTA
//               waiting for the longest row; and the heads of a position,
//               neighbours in memory, are read at about the same time. Every
//               warp works the cut out for itself from the rows' lengths. A
//               second launch joins the items' runs.
//   kClustered  An item is a cluster's: each CTA takes an equal run, and they
//               join through distributed shared memory. One launch, for short
//               contexts, where the second one would be most of the time.
//   kRuns       A CTA takes one run of kRun pieces at least (or, with room for
//               one part only, the item): for rows too many to be dealt.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(Shape<T, HD, NT>::warps * 32, Shape<T, HD, NT>::ctas)
paged_attn_kernel(const AttnArgs a) {
  using S = Shape<T, HD, NT>;
  extern __shared__ __align__(16) unsigned char sm[];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, kt = a.n_kv * a.tiles;

  int row, len, u;                  // the current row, its positions and pieces
  if (a.mode == kDealt) {
    for (row = blockIdx.x; row < a.rows; row += gridDim.x)
      if (length_of(a, row) == 0) clear_heads<T>(a, row, 0, a.n_q);
    const unsigned group = blockIdx.x / kt;
    const int i = blockIdx.x - group * kt;
    const int per = (a.rows + 31) / 32, r0 = min(lane * per, a.rows), r1 = min(r0 + per, a.rows);
    int sum = 0, most = 0, last_len = 0;
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {
      last_len = length_of(a, r);
      const int n = pieces_of(last_len);
      sum += n;
      most = max(most, n);
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned total = __shfl_sync(~0u, upto, 31);
    most = __reduce_max_sync(~0u, most);
    if (total == 0) return;
    // Group g takes pieces floor(g total / G) to floor((g + 1) total / G), so
    // piece x is group floor(((x + 1) G - 1) / total)'s. u pieces meet at most
    // ceil((u - 1) G / total) + 1 groups: G is kept so low that this is at most
    // a.parts. (The host sees to it that these products stay below 2^32.)
    unsigned G = min((unsigned)(gridDim.x / kt), total);
    if (most > 1) G = min(G, max(1u, (a.parts - 1) * total / (most - 1)));
    if (group >= G) return;
    int w = (int)(group * total / G);              // this group's pieces
    const int w1 = (int)((group + 1) * total / G);
    const int owner = __ffs(__ballot_sync(~0u, upto > w)) - 1;
    row = owner * per;
    int base = __shfl_sync(~0u, upto - sum, owner);   // where the row's pieces begin
    len = per == 1 ? __shfl_sync(~0u, last_len, owner) : length_of(a, row);
    u = pieces_of(len);
    for (;;) {
      while (base + u <= w) {
        base += u;
        if (++row >= a.rows) return;
        len = length_of(a, row);
        u = pieces_of(len);
      }
      const int off = w - base, n = min(u - off, w1 - w);
      const int first = (int)(((base + 1u) * G - 1) / total), last = (int)(((unsigned)(base + u) * G - 1) / total);
      const int part = (int)group - first;
      // Lengths that somebody changes while the kernel runs make the warps' cuts
      // disagree; the result is then anything, but nothing outside is touched.
      if (off < 0 || part < 0 || part >= a.parts) return;
      attend<T, HD, NT>(a, sm, row, i / a.tiles, i % a.tiles, off * kPiece, min(len, (off + n) * kPiece), part,
                        last - first + 1);
      w += n;
      if (w >= w1) return;
      __syncthreads();              // the ring is free again
    }
  }
  const int run_part = blockIdx.x % a.parts, item = blockIdx.x / a.parts, i = item % kt;
  row = item / kt;
  len = length_of(a, row);
  if (len <= 0) {
    const int tile = i % a.tiles;
    if (len == 0 && run_part == 0)
      clear_heads<T>(a, row, i / a.tiles * a.group + tile * S::heads, min(S::heads, a.group - tile * S::heads));
    if (a.mode == kClustered) { cluster_sync(); cluster_sync(); }
    return;
  }
  u = pieces_of(len);
  int run = (u - 1) / a.parts + 1;
  if (a.mode == kRuns && a.parts > 1) run = max(kRun, run);
  const int w = min(run_part * run, u), w1 = min(w + run, u);
  // a cluster's CTA without a run of its own still takes part in the join
  if (w >= w1 && a.mode != kClustered) return;
  attend<T, HD, NT>(a, sm, row, i / a.tiles, i % a.tiles, min(len, w * kPiece), min(len, w1 * kPiece), run_part,
                    a.mode == kClustered ? a.parts : (u - 1) / run + 1);
  if (a.mode == kClustered) cluster_sync();        // the others may still be reading here
}

// Joins the runs of a row: a block per (row, query head), the runs dealt to
// its 8 warps, each lane four (or eight) elements of the head. Its time is the
// latency of its loads, so the first 4 runs of every warp are loaded beside
// the runs' maxima and sums, before it is known how many runs there are (what
// lies behind them in the workspace is not used).
// One warp to a head where heads are many, and blocks small enough to be
// resident before the first kernel ends, measured no better (59.2 us for 59.5 of
// 32 rows, 50.2 for 49.2 of one long row): most of the 4 us are the first
// kernel's end becoming known.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join_kernel(const AttnArgs a) {
  __shared__ float sw[kMaxParts], red[kJoinWarps][256], total;
  const int row = blockIdx.x / a.n_q, h = blockIdx.x % a.n_q;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = length_of(a, row);             // written before the launch that this one follows
  const long long base = ((long long)row * a.n_q + h) * a.parts;
  // every block waits, those without work too: what follows this launch in
  // the stream relies on the first kernel's results being there
  pdl_wait();
  pdl_launch();
  if (len <= 0) return;
  float2 ml[kMaxParts / 32];
#pragma unroll
  for (int j = 0; j < kMaxParts / 32; ++j) {
    const int p = j * 32 + lane;
    ml[j] = p < a.parts ? a.part_ml[base + p] : make_float2(0.f, 0.f);
  }
  float4 x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = warp + j * kJoinWarps;
    x[j] = p < a.parts && 4 * lane < a.hd ? *reinterpret_cast<const float4*>(a.part_o + (base + p) * a.hd + 4 * lane)
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int n = 0;                                     // runs: the last one is marked
#pragma unroll
  for (int j = 0; j < kMaxParts / 32; ++j) {
    const unsigned marks = __ballot_sync(~0u, __float_as_uint(ml[j].y) >> 31);
    if (n == 0 && marks) n = j * 32 + __ffs(marks);
  }
  if (n <= 1) return;                            // its only run has written the result
  float m = -FLT_MAX;
#pragma unroll
  for (int j = 0; j < kMaxParts / 32; ++j) {
    ml[j] = j * 32 + lane < n ? make_float2(ml[j].x, fabsf(ml[j].y)) : make_float2(-FLT_MAX, 0.f);
    m = fmaxf(m, ml[j].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (warp == 0) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxParts / 32; ++j) {
      const float f = ex2(ml[j].x - m);
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
    auto add = [&](int p, const float4& v) {
      const float f = sw[p];
      acc[0] = fmaf(f, v.x, acc[0]); acc[1] = fmaf(f, v.y, acc[1]);
      acc[2] = fmaf(f, v.z, acc[2]); acc[3] = fmaf(f, v.w, acc[3]);
    };
    int p = warp;
    if (d < 128) {
#pragma unroll
      for (int j = 0; j < 4; ++j, p += kJoinWarps)
        if (p < n) add(p, x[j]);
    }
#pragma unroll 6
    for (; p < n; p += kJoinWarps) add(p, *reinterpret_cast<const float4*>(a.part_o + (base + p) * a.hd + d));
    *reinterpret_cast<float4*>(&red[warp][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.hd; d += kJoinWarps * 32) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) y += red[w][d];
    store1<T>(a.out, row * a.ldo + (long long)h * a.hd + d, total == 0.f ? 0.f : y / total);
  }
}

// ---- host side ---------------------------------------------------------------

int head_tile(int dtype, int hd, int group) {
  return dtype != MOE_DTYPE_F32 && hd <= 128 && group > 8 ? 16 : 8;
}

// The split of a call, from what the host knows of it, and the parts that a
// row's head may have. Short contexts: clusters of as many CTAs as bring their
// number to 200, one where the items alone are that many (clusters are slow to
// place: 16 rows of 1024 positions take 10.3 us in 256 CTAs, 15.0 in 512; 64
// rows 25 us in 256, 34 in 1024).
struct Split { int mode, parts; };
Split split_of(long long items, int rows, int max_kv) {
  const int pieces = (max_kv - 1) / kPiece + 1;
  if (pieces <= kShort) {
    int n = 1;
    while (n < kCluster && n < pieces && items * n < 200) n *= 2;
    return {n > 1 ? kClustered : kRuns, n};
  }
  if (rows > kDealtRows) {
    // The more rows, the fewer parts each: they fill the GPU, and a part for
    // every run of each row's context costs workspace and the second launch
    // (8192 rows of one prompt, 32 heads of 128: 16 parts 2.2 GB and 7.9 ms, 2
    // parts 0.27 GB and 6.0 ms; one row of 131072 among 600 short ones: 128 parts
    // 1.3 GB and 0.62 ms, 27 parts 0.27 GB and 0.26 ms).
    const int runs = (pieces - 1) / kRun + 1, most = kRowParts / rows;
    if (most <= 1) return {kRuns, 1};
    const int n = most < kMaxParts ? most : kMaxParts;
    return {kRuns, runs < n ? runs : n};
  }
  return {kDealt, pieces < kMaxParts ? pieces : kMaxParts};
}

int sm_count(int device) {
  static std::atomic<int> count[64];
  if (device < 0 || device >= 64) return 148;
  int n = count[device].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) n = 148;
    count[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <typename T, int HD, int NT>
cudaError_t launch_attn(AttnArgs a, int max_kv, int device, cudaStream_t st) {
  using S = Shape<T, HD, NT>;
  static std::atomic<unsigned long long> ready{0};       // devices whose limit is raised
  const unsigned long long bit = 1ull << (device & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<T, HD, NT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return e;
    if (device < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  const long long items = (long long)a.rows * a.n_kv * a.tiles, sms = sm_count(device);
  long long grid = items * a.parts;
  if (a.mode == kDealt) {
    // as many groups as the GPU holds at a time, if the rows have parts and
    // pieces for them
    const long long kt = (long long)a.n_kv * a.tiles, fit = sms * S::ctas / kt, pieces = (max_kv - 1) / kPiece + 1;
    long long groups = fit < a.rows * (a.parts - 1ll) ? fit : a.rows * (a.parts - 1ll);
    if (groups > a.rows * pieces) groups = a.rows * pieces;
    if (groups > 1023) groups = 1023;
    grid = (groups > 1 ? groups : 1) * kt;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(S::warps * 32); cfg.dynamicSmemBytes = S::smem; cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.mode == kClustered) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = a.parts; at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<T, HD, NT>, a);
  if (e != cudaSuccess || a.mode == kClustered || a.parts == 1) return e;
  return launch_pdl(paged_attn_join_kernel<T>, dim3((unsigned)a.rows * (unsigned)a.n_q), dim3(kJoinWarps * 32), 0, st, a);
}

template <typename T>
cudaError_t launch_type(const AttnArgs& a, int tile, int max_kv, int device, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (tile == 16 && a.hd <= 64) return launch_attn<T, 64, 2>(a, max_kv, device, st);
    if (tile == 16 && a.hd <= 96) return launch_attn<T, 96, 2>(a, max_kv, device, st);
    if (tile == 16) return launch_attn<T, 128, 2>(a, max_kv, device, st);
  }
  if (a.hd <= 64) return launch_attn<T, 64, 1>(a, max_kv, device, st);
  if (a.hd <= 96) return launch_attn<T, 96, 1>(a, max_kv, device, st);
  if (a.hd <= 128) return launch_attn<T, 128, 1>(a, max_kv, device, st);
  return launch_attn<T, 256, 1>(a, max_kv, device, st);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_paged_attention_workspace(int rows, int n_q, const MoeKvCache* cache, int max_kv) {
  if (at::check_cache(cache, "moe_paged_attention_workspace")) return 0;
  if (rows < 1 || n_q < 1 || n_q % cache->n_kv || max_kv < 1) return 0;
  const int group = n_q / cache->n_kv, ht = head_tile(cache->dtype, cache->head_dim, group);
  const long long items = (long long)rows * cache->n_kv * ((group + ht - 1) / ht);
  const Split sp = split_of(items, rows, max_kv);
  if (sp.parts == 1 || sp.mode == kClustered) return 0;
  return (size_t)rows * n_q * sp.parts * (sizeof(float2) + sizeof(float) * cache->head_dim) + 16;
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
  if (n_q > 32768) return at::fail(MOE_ERR_UNSUPPORTED, "%s: %d query heads (at most 32768)", who, n_q);
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
  const long long nq = (long long)n_q * hd;
  if (!(out == q && ldo == ldq) && at::overlap(out, ldo, nq, es, q, ldq, nq, es, rows))
    return at::fail(MOE_ERR_INVALID, "%s: out overlaps q without being q", who);
  const int group = n_q / cache->n_kv, ht = head_tile(cache->dtype, hd, group);
  AttnArgs a{};
  a.tiles = (group + ht - 1) / ht;
  const long long items = (long long)rows * cache->n_kv * a.tiles;
  const Split sp = split_of(items, rows, max_kv);
  a.parts = sp.parts;
  a.mode = sp.mode;
  // where pieces are dealt out, their number times that of the groups (fewer
  // than 1024) has 32 bits
  const long long pieces = (long long)max_pages * cache->page_size / kPiece + 1;
  if (a.mode == kDealt && rows * pieces > INT32_MAX / 1024) a.mode = kRuns;
  if (items * a.parts > INT32_MAX || (long long)rows * n_q > INT32_MAX)
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
  if (cache->dtype == MOE_DTYPE_BF16) e = launch_type<__nv_bfloat16>(a, ht, max_kv, on.device(), st);
  else if (cache->dtype == MOE_DTYPE_F16) e = launch_type<__half>(a, ht, max_kv, on.device(), st);
  else e = launch_type<float>(a, ht, max_kv, on.device(), st);
  return at::launched(e, who);
}
