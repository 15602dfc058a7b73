// kv_plan.cu — moe_kv_plan_dev: the block tables and slot maps of a paged
// key-value cache, built on the GPU from the sequences' lengths, so that a
// captured decode step needs no host in between (and no host copy of any
// length).
//
// With P = page_size: sequence s holds ceil(past_s/P) pages and needs
// ceil((past_s + new_s)/P). The missing pages come off the free list in
// sequence order, so page j of sequence s is free[head + start_s + (j - held_s)]
// with start_s the exclusive sum of the earlier sequences' missing pages. Row i
// belongs to the sequence whose inclusive sum of new lengths first exceeds i.
//
// Nothing here is bound by bytes (a 32-sequence decode step reads and writes
// about a kilobyte): the time is a launch and a chain of dependent loads. So
// every CTA scans all lengths for itself in shared memory rather than waiting
// for another CTA's scan, and rows and pages are then spread evenly over all
// threads, which find their sequences by bisection: a long prompt costs no
// single warp more than the others.
//
// kv_len may be past_len and free_head_out free_head. With one CTA a barrier
// between reading and writing does for that; with several, another launch of
// one CTA writes them when all have read.
#include "attn.cuh"

namespace moe {
namespace {

constexpr int kMaxSeqs = 16384;      // 12 bytes of shared memory each
constexpr int kMaxThreads = 512;
constexpr size_t kStatic = 2 * 32 * sizeof(int);   // the kernel's own shared memory, which counts too

struct PlanArgs {
  const int *past_len, *new_len, *free_pages, *free_head;
  int *table, *kv_len, *row_seq, *row_pos, *row_slot, *head_out, *status;
  long long table_stride;
  int n_seq, page_size, n_pages, n_free, max_pages, row_cap;
  int quads;              // rows are taken four at a time
  int plan, sums;         // whether this launch writes pages and rows; kv_len, free_head_out and status
  at::FastDiv page;
};

// min(a + b, INT_MAX) for a, b >= 0 (associative, so it can be scanned)
__device__ __forceinline__ int sat_add(int a, int b) {
  const unsigned s = (unsigned)a + (unsigned)b;
  return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}

__device__ __forceinline__ int pages_of(const PlanArgs& a, int len) {
  const int n = (int)a.page.div((unsigned)len);
  return min(n + (n * a.page_size < len), a.max_pages);
}

// first s with end[s] > i; the caller knows that one exists
__device__ __forceinline__ int owner_of(const int* end, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (end[mid] > i) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kMaxThreads) kv_plan_kernel(const PlanArgs a) {
  pdl_wait();
  pdl_launch();
  extern __shared__ int sm[];
  __shared__ int warp_rows[32], warp_pages[32];
  static_assert(sizeof(warp_rows) + sizeof(warp_pages) == kStatic, "");
  int *past = sm, *row_end = sm + a.n_seq, *page_end = sm + 2 * a.n_seq;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = gridDim.x, cta = blockIdx.x;

  // each thread sums a run of consecutive sequences, the block scans the sums
  const int per = (a.n_seq + nt - 1) / nt, s0 = min(tid * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
  int rows = 0, pages = 0;
  for (int s = s0; s < s1; ++s) {
    const int p = a.past_len ? max(a.past_len[s], 0) : 0;
    const int n = min(max(a.new_len[s], 0), 0x7fffffff - p);
    past[s] = p;
    rows = sat_add(rows, n);
    pages += pages_of(a, p + n) - pages_of(a, p);
    row_end[s] = rows;
    page_end[s] = pages;
  }
  int head = a.free_head ? *a.free_head : 0;
  head = min(max(head, 0), a.n_free);
  int r = rows, g = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int r2 = __shfl_up_sync(~0u, r, o), g2 = __shfl_up_sync(~0u, g, o);
    if (lane >= o) { r = sat_add(r, r2); g += g2; }
  }
  if (lane == 31) { warp_rows[warp] = r; warp_pages[warp] = g; }
  __syncthreads();
  int r0 = 0, g0 = 0, all_rows = 0, all_pages = 0;
  for (int w = 0; w < nt / 32; ++w) {
    if (w == warp) { r0 = all_rows; g0 = all_pages; }
    all_rows = sat_add(all_rows, warp_rows[w]);
    all_pages += warp_pages[w];
  }
  const int r1 = __shfl_up_sync(~0u, r, 1), g1 = __shfl_up_sync(~0u, g, 1);
  if (lane) { r0 = sat_add(r0, r1); g0 += g1; }
  for (int s = s0; s < s1; ++s) { row_end[s] = sat_add(row_end[s], r0); page_end[s] += g0; }
  __syncthreads();

  const unsigned first = cta * nt + tid, step = ctas * nt;
  const int taken = min(all_pages, a.n_free - head);
  if (a.sums && cta == 0) {
    if (a.kv_len)
      for (int s = tid; s < a.n_seq; s += nt) a.kv_len[s] = past[s] + (row_end[s] - (s ? row_end[s - 1] : 0));
    if (tid == 0) {
      if (a.head_out) *a.head_out = head + taken;
      if (a.status) { a.status[0] = all_rows; a.status[1] = all_pages; a.status[2] = taken; }
    }
  }
  if (!a.plan) return;
  for (unsigned j = first; j < (unsigned)all_pages; j += step) {
    const int s = owner_of(page_end, a.n_seq, (int)j), start = s ? page_end[s - 1] : 0;
    a.table[s * a.table_stride + pages_of(a, past[s]) + ((int)j - start)] = (int)j < taken ? a.free_pages[head + j] : -1;
  }
  // row i of sequence s
  auto row_of = [&](int i, int s, int& pos, int& slot) {
    pos = past[s] + (i - (s ? row_end[s - 1] : 0));
    const int pi = (int)a.page.div((unsigned)pos), held = pages_of(a, past[s]);
    int pg = -1;
    if (pi < a.max_pages) {
      if (pi < held) pg = a.table[s * a.table_stride + pi];
      else {
        const int j = (s ? page_end[s - 1] : 0) + (pi - held);
        if (j < taken) pg = a.free_pages[head + j];
      }
    }
    slot = pg >= 0 && pg < a.n_pages ? pg * a.page_size + (pos - pi * a.page_size) : -1;
  };
  if (!a.quads) {
    for (unsigned i = first; i < (unsigned)a.row_cap; i += step) {
      int s = -1, pos = -1, slot = -1;
      if (i < (unsigned)all_rows) {
        s = owner_of(row_end, a.n_seq, (int)i);
        row_of((int)i, s, pos, slot);
      }
      a.row_seq[i] = s;
      a.row_pos[i] = pos;
      a.row_slot[i] = slot;
    }
    return;
  }
  // Four consecutive rows a thread: one search for the first of them, then on
  // from sequence to sequence.
  for (unsigned i0 = 4 * first; i0 < (unsigned)a.row_cap; i0 += 4 * step) {
    int seq[4] = {-1, -1, -1, -1}, pos[4] = {-1, -1, -1, -1}, slot[4] = {-1, -1, -1, -1};
    if (i0 < (unsigned)all_rows) {
      int s = owner_of(row_end, a.n_seq, (int)i0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = (int)(i0 + k);
        if (i0 + k >= (unsigned)all_rows) break;
        while (row_end[s] <= i) ++s;
        seq[k] = s;
        row_of(i, s, pos[k], slot[k]);
      }
    }
    if (i0 + 4 <= (unsigned)a.row_cap) {
      *reinterpret_cast<int4*>(a.row_seq + i0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
      *reinterpret_cast<int4*>(a.row_pos + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.row_slot + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < (unsigned)a.row_cap) { a.row_seq[i0 + k] = seq[k]; a.row_pos[i0 + k] = pos[k]; a.row_slot[i0 + k] = slot[k]; }
    }
  }
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_kv_plan_dev(const int* past_len, const int* new_len, int n_seq, int page_size, int n_pages,
                               const int* free_pages, int n_free, const int* free_head, int* block_table,
                               int max_pages, int* kv_len, int* row_seq, int* row_pos, int* row_slot, int row_cap,
                               int* free_head_out, int* status, void* stream) {
  static const char who[] = "moe_kv_plan_dev";
  if (n_seq < 0 || row_cap < 0 || n_free < 0) return at::fail(MOE_ERR_INVALID, "%s: negative size", who);
  if (n_seq > kMaxSeqs) return at::fail(MOE_ERR_UNSUPPORTED, "%s: %d sequences (at most %d)", who, n_seq, kMaxSeqs);
  if (page_size < 1 || n_pages < 1 || max_pages < 1)
    return at::fail(MOE_ERR_INVALID, "%s: page_size %d, n_pages %d, max_pages %d", who, page_size, n_pages, max_pages);
  if ((long long)n_pages * page_size > INT32_MAX)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 slots", who);
  if ((long long)n_seq * max_pages > INT32_MAX)
    return at::fail(MOE_ERR_UNSUPPORTED, "%s: block table of more than 2^31 - 1 entries", who);
  if (n_seq && (!new_len || !block_table)) return at::fail(MOE_ERR_INVALID, "%s: new_len and block_table are needed", who);
  if (n_free && !free_pages) return at::fail(MOE_ERR_INVALID, "%s: n_free without free_pages", who);
  if (row_cap && (!row_seq || !row_pos || !row_slot))
    return at::fail(MOE_ERR_INVALID, "%s: row_seq, row_pos and row_slot are needed", who);
  const void* any = n_seq ? (const void*)block_table : row_cap ? (const void*)row_seq
                  : free_head_out ? (const void*)free_head_out : (const void*)status;
  if (!any) return MOE_OK;
  at::OnDeviceOf on;
  int rc = on.enter(any, who);
  if (rc) return rc;
  PlanArgs a{};
  a.past_len = past_len; a.new_len = new_len; a.free_pages = free_pages; a.free_head = free_head;
  a.table = block_table; a.kv_len = kv_len; a.row_seq = row_seq; a.row_pos = row_pos; a.row_slot = row_slot;
  a.head_out = free_head_out; a.status = status; a.table_stride = max_pages;
  a.n_seq = n_seq; a.page_size = page_size; a.n_pages = n_pages; a.n_free = n_free; a.max_pages = max_pages;
  a.row_cap = row_cap; a.page = at::FastDiv((unsigned)page_size);
  // one row a thread up to 2048 (latency), four in large plans
  a.quads = row_cap > 2048 && ((uintptr_t)row_seq | (uintptr_t)row_pos | (uintptr_t)row_slot) % 16 == 0;
  const int work = n_seq > row_cap ? n_seq : row_cap, each = kMaxThreads * (a.quads ? 4 : 1);
  const int threads = work <= 256 ? 256 : kMaxThreads;
  const int ctas = work <= 2 * kMaxThreads ? 1 : work / each < 148 ? (work + each - 1) / each : 148;
  const bool in_place = ctas > 1 && ((kv_len && (kv_len == past_len || kv_len == new_len)) || (free_head_out && free_head_out == free_head));
  const size_t smem = sizeof(int) * 3 * (size_t)n_seq;
  if (smem + kStatic > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(sizeof(int) * 3 * kMaxSeqs));
    if (e != cudaSuccess) return at::fail(MOE_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  }
  a.plan = 1;
  a.sums = !in_place;
  cudaError_t e = launch_pdl(kv_plan_kernel, dim3(ctas), dim3(threads), smem, (cudaStream_t)stream, a);
  if (e == cudaSuccess && in_place) {
    a.plan = 0;
    a.sums = 1;
    e = launch_pdl(kv_plan_kernel, dim3(1), dim3(threads), smem, (cudaStream_t)stream, a);
  }
  return at::launched(e, who);
}
