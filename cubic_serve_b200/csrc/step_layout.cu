// The layout of a step from the lengths of its requests: block table, slots, positions and the row blocks of the attention.
//
// Request i has start[i] tokens in the cache and brings count[i]; its row of the block table holds the first held[i] pages.  With
//   need[i] = max(0, ceil((start[i] + count[i]) / 16) - held[i]),  off = exclusive sum of need,  row0 = exclusive sum of count
// it takes pages[off[i] .. off[i] + need[i]) behind those it holds, and its token j (row row0[i] + j of the step) is at
//   position start[i] + j,  slot 16 page(position / 16) + position % 16.
// A row block is up to `block` neighbouring tokens of one request.
//
// Bound by latency: 256 decoding requests are 4 KB in and 6 KB out.  One launch; every CTA makes the three sums of all requests for itself (a few per
// thread) and keeps them in shared memory, so that no CTA waits for another; a page that is taken in this step is read from the list
// and not from the table, which another CTA may be writing.  Owners are found by bisection, four outputs a thread in one 16-byte store.
// 256 decoding requests take 4.6 us, 37 portions of up to 220 tokens 4.3, 300 of up to 700 5.6 (their 3.5 MB would take 0.5): a launch, four trips to memory in
// a row (ids and lengths; table or page; store) and the scan.
#include "ptx.cuh"
#include "launch.cuh"

namespace cb {

static constexpr int kLayoutThreads = 256;
static constexpr int kLayoutMaxRequests = 4096;
static constexpr int kLayoutPage = 16;
static constexpr int kLayoutMost = 1 << 29;

}  // namespace cb

// Packed by ops/native.py::STEP_LAYOUT.
struct CbStepLayout {
  const int* request;        // [n] row of the block table
  const int* start;          // [n] tokens before the step
  const int* count;          // [n] new tokens
  const int* held;           // [n] pages in the row, null: ceil(start / 16)
  const int* pages;          // [num_pages] what requests take, in their order
  int* table;                // [table_rows, width], row stride ld
  int* positions; int* slots;                                // [cap_tokens]
  int* rb_req; int* rb_qstart; int* rb_qcount; int* rb_ctx;  // [cap_blocks]
  int* row0;                 // [n]
  long long* logit_rows;     // [n] last row of the request, -1: no new tokens
  int* totals;               // [4] tokens, row blocks, pages taken, what went wrong (kLayout... bits)
  int n, num_pages, table_rows, width, ld, block;
  int cap_tokens, cap_blocks;            // rows that may be written
  int pad;                               // rows behind the last token / row block up to here are padding
};

namespace cb {

enum { kLayoutNoPages = 1, kLayoutTooLong = 2, kLayoutBadRequest = 4, kLayoutTooMany = 8 };

struct LayoutShared {
  int *rows, *blocks, *taken;            // [n + 1] exclusive sums
  int *start, *request, *held;           // [n]
};

// Last i with upto[i] <= v: the owner of entry v (entries of empty requests have none).
__device__ __forceinline__ int owner(const int* upto, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (upto[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// Sums that stop at kLayoutMost: what is behind it lies outside every buffer, and nothing overflows.
__device__ __forceinline__ int3 add(int3 a, int3 b) {
  return make_int3(min(a.x + b.x, kLayoutMost), min(a.y + b.y, kLayoutMost), min(a.z + b.z, kLayoutMost));
}

__device__ __forceinline__ void store4(int* p, int i, int cap, const int (&v)[4]) {
  if (i + 4 <= cap && (reinterpret_cast<uintptr_t>(p + i) & 15) == 0) {
    *reinterpret_cast<int4*>(p + i) = make_int4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j < cap) p[i + j] = v[j];
}

__global__ void __launch_bounds__(kLayoutThreads)
step_layout_kernel(const CbStepLayout p) {
  extern __shared__ int sm[];
  __shared__ int3 warp_sum[kLayoutThreads / 32];
  __shared__ int bad;
  const int n = p.n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  LayoutShared s;
  s.rows = sm; s.blocks = s.rows + n + 1; s.taken = s.blocks + n + 1;
  s.start = s.taken + n + 1; s.request = s.start + n; s.held = s.request + n;
  if (tid == 0) bad = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();

  // a thread's run of requests, then the sums before it
  const int per = (n + kLayoutThreads - 1) / kLayoutThreads, lo = min(n, tid * per), hi = min(n, lo + per);
  int3 sum = make_int3(0, 0, 0);
  for (int i = lo; i < hi; ++i) {
    const int start = min(max(0, p.start[i]), kLayoutMost), c = min(max(0, p.count[i]), kLayoutMost);
    const int held = max(0, p.held ? p.held[i] : (start + kLayoutPage - 1) / kLayoutPage), pages = (start + c + kLayoutPage - 1) / kLayoutPage;
    int req = p.request[i];
    const int wrong = (req < 0 || req >= p.table_rows ? kLayoutBadRequest : 0) | (pages > p.width || held > p.width ? kLayoutTooLong : 0);
    if (wrong) { atomicOr(&bad, wrong); req = -1; }                  // no pages, no slots, nothing for the attention to read
    s.start[i] = start; s.request[i] = req; s.held[i] = held;
    s.rows[i] = c; s.blocks[i] = (c + p.block - 1) / p.block; s.taken[i] = wrong ? 0 : max(0, pages - held);
    sum = add(sum, make_int3(s.rows[i], s.blocks[i], s.taken[i]));
  }
  int3 inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int3 before = make_int3(__shfl_up_sync(0xffffffffu, inc.x, o), __shfl_up_sync(0xffffffffu, inc.y, o), __shfl_up_sync(0xffffffffu, inc.z, o));
    if (lane >= o) inc = add(inc, before);
  }
  // the sum before the thread's own run
  int3 run = make_int3(__shfl_up_sync(0xffffffffu, inc.x, 1), __shfl_up_sync(0xffffffffu, inc.y, 1), __shfl_up_sync(0xffffffffu, inc.z, 1));
  if (lane == 0) run = make_int3(0, 0, 0);
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int3 total = make_int3(0, 0, 0);
#pragma unroll
  for (int w = 0; w < kLayoutThreads / 32; ++w) {
    if (w == warp) run = add(total, run);
    total = add(total, warp_sum[w]);
  }
  for (int i = lo; i < hi; ++i) {
    const int3 mine = make_int3(s.rows[i], s.blocks[i], s.taken[i]);
    s.rows[i] = run.x; s.blocks[i] = run.y; s.taken[i] = run.z;
    run = add(run, mine);
  }
  if (tid == 0) { s.rows[n] = total.x; s.blocks[n] = total.y; s.taken[n] = total.z; }
  __syncthreads();

  const int tokens = min(total.x, p.cap_tokens), blocks = min(total.y, p.cap_blocks), taken = min(total.z, p.num_pages);
  const int rows_end = min(max(tokens, p.pad), p.cap_tokens), blocks_end = min(max(blocks, p.pad), p.cap_blocks);
  const int u0 = (rows_end + 3) >> 2, u1 = u0 + ((blocks_end + 3) >> 2), u2 = u1 + taken, u3 = u2 + n;
  for (int u = blockIdx.x * kLayoutThreads + tid; u < u3; u += gridDim.x * kLayoutThreads) {
    if (u < u0) {                                                    // four tokens
      int pos[4], slot[4];
      const int t = u << 2;
      int i = t < tokens ? owner(s.rows, n, t) : n;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pos[j] = 0; slot[j] = -1;
        if (t + j >= tokens) continue;
        while (t + j >= s.rows[i + 1]) ++i;
        pos[j] = s.start[i] + (t + j - s.rows[i]);
        const int pg = pos[j] / kLayoutPage, req = s.request[i], take = s.taken[i] + (pg - s.held[i]);
        if (req < 0) continue;
        int page = -1;
        if (pg < s.held[i]) page = p.table[static_cast<size_t>(req) * p.ld + pg];
        else if (take < p.num_pages) page = p.pages[take];
        if (page >= 0 && page < (1 << 27)) slot[j] = page * kLayoutPage + (pos[j] % kLayoutPage);
      }
      store4(p.positions, t, rows_end, pos);
      store4(p.slots, t, rows_end, slot);
    } else if (u < u1) {                                             // four row blocks
      int req[4], first[4], num[4], ctx[4];
      const int b = (u - u0) << 2;
      int i = b < blocks ? owner(s.blocks, n, b) : n;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        req[j] = 0; first[j] = b + j; num[j] = 0; ctx[j] = 0;
        if (b + j >= blocks) continue;
        while (b + j >= s.blocks[i + 1]) ++i;
        const int f = (b + j - s.blocks[i]) * p.block, c = s.rows[i + 1] - s.rows[i];
        req[j] = s.request[i]; first[j] = s.rows[i] + f; num[j] = min(c - f, p.block); ctx[j] = s.start[i] + f + 1;
        // what has no row, got no pages or lies behind the rows that are written attends to nothing
        if (req[j] < 0 || (s.taken[i + 1] > s.taken[i] && s.taken[i + 1] > p.num_pages) || first[j] + num[j] > tokens) { req[j] = 0; num[j] = 0; ctx[j] = 0; }
      }
      store4(p.rb_req, b, blocks_end, req);
      store4(p.rb_qstart, b, blocks_end, first);
      store4(p.rb_qcount, b, blocks_end, num);
      store4(p.rb_ctx, b, blocks_end, ctx);
    } else if (u < u2) {                                             // a page that is taken
      const int k = u - u1, i = owner(s.taken, n, k), at = s.held[i] + (k - s.taken[i]);
      p.table[static_cast<size_t>(s.request[i]) * p.ld + at] = p.pages[k];
    } else {
      const int i = u - u2;
      p.row0[i] = s.rows[i];
      const int last = s.rows[i + 1] - 1;
      p.logit_rows[i] = s.rows[i + 1] > s.rows[i] && last < tokens ? last : -1;
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.totals[0] = total.x; p.totals[1] = total.y; p.totals[2] = total.z;
    p.totals[3] = bad | (total.z > p.num_pages ? kLayoutNoPages : 0) | (total.x > p.cap_tokens || total.y > p.cap_blocks ? kLayoutTooMany : 0);
  }
}

}  // namespace cb

extern "C" int cb_step_layout(const CbStepLayout* p, void* stream) {
  using namespace cb;
  if (p->cap_tokens > kLayoutMost / 2 || p->cap_blocks > kLayoutMost / 2 || p->num_pages > kLayoutMost / 2) return -11;
  if (p->n < 0 || p->n > kLayoutMaxRequests || p->block < 1 || p->pad > p->cap_tokens || p->pad > p->cap_blocks || p->ld < p->width) return -10;
  const size_t smem = static_cast<size_t>(6 * p->n + 3) * sizeof(int);
  static bool ready[64] = {};            // once a device, whatever the size: the kernel's own arrays count towards the usual 48 KB too
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev]))
    e = cudaFuncSetAttribute(step_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (6 * kLayoutMaxRequests + 3) * sizeof(int));
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 64) ready[dev] = true;
  const int units = p->cap_tokens / 4 + p->cap_blocks / 4 + 2 + p->num_pages + p->n, grid = min(296, (units + kLayoutThreads - 1) / kLayoutThreads);
  return static_cast<int>(launch(step_layout_kernel, dim3(grid), dim3(kLayoutThreads), smem, static_cast<cudaStream_t>(stream), *p));
}
