// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + scale[s] (x[t] A[s]^T) B[s]^T,  s = adapter of row t (none: out[t] = y[t]).
// A projection made of sections (q | k | v, gate | up) has an A of its own for each: A[s] stacks them, and the columns of section j see
// ranks [j rank, (j + 1) rank).
//
// Three kernels.  `adapter_rows_kernel` sorts a step's rows by adapter, once for all projections of all layers.  `adapter_down_kernel`
// makes h = scale x A^T of the sorted rows, `adapter_up_kernel` adds h B^T.  A work item is up to 64 rows of one adapter.
//
// Bound by memory: with few rows by A and B of the adapters in use, with many by y and out.  The products run on
// mma.sync m16n8k16 with operands that go from global memory to registers: rank 16 makes 16 products of every byte of x, far from
// what would keep tensor memory busy, and a stage of shared memory would add a round trip to a chain of two short kernels.
#include "ptx.cuh"
#include "mma.cuh"
#include "launch.cuh"

namespace cb {

static constexpr int kAdapterItemRows = 64;
static constexpr int kAdapterMaxSlots = 1023;
static constexpr int kAdapterMaxRows = 65535;
static constexpr int kAdapterSections = 4;
static constexpr int kSortThreads = 1024;
static constexpr int kAdapterThreads = 256;

// ------------------------------------------------------------------ rows by adapter
// order[]: the step's rows by adapter, a row's place among its adapter's by its index; rows without one last.
// items[]: [0] = count, then {adapter (-1: none), first place, rows}.
// One CTA: a warp counts the adapters of its share of the rows, the counts become places, a second look at the ids fills them.  8192 rows
// are two rounds of 8 steps a warp.
__global__ void __launch_bounds__(kSortThreads)
adapter_rows_kernel(const int* __restrict__ ids, int rows, int slots, int* __restrict__ order, int* __restrict__ items) {
  extern __shared__ unsigned short cnt[];                             // [32 warps][buckets]
  __shared__ int warp_rows[32], warp_items[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, buckets = slots + 1;
  const int share = (((rows + 31) >> 5) + 31) & ~31, lo = min(rows, warp * share), hi = min(rows, lo + share);
  for (int i = tid; i < 32 * buckets; i += kSortThreads) cnt[i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  unsigned short* mine = cnt + warp * buckets;
  for (int r = lo; r < hi; r += 32) {
    const int row = r + lane;
    int b = -1;
    if (row < hi) { b = ids[row]; if (b < 0 || b >= slots) b = slots; }
    const uint32_t same = __match_any_sync(0xffffffffu, b);
    if (b >= 0 && lane == __ffs(same) - 1) mine[b] = static_cast<unsigned short>(mine[b] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  // counts of the warps before, rows and items of the buckets before
  int n = 0;
  if (tid < buckets)
    for (int w = 0; w < 32; ++w) {
      const int c = cnt[w * buckets + tid];
      cnt[w * buckets + tid] = static_cast<unsigned short>(n);
      n += c;
    }
  const int nt = (n + kAdapterItemRows - 1) / kAdapterItemRows;
  int at = n, it = nt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, at, o), b = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) { at += a; it += b; }
  }
  if (lane == 31) { warp_rows[warp] = at; warp_items[warp] = it; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { at += warp_rows[w]; it += warp_items[w]; }
  at -= n;
  if (tid < buckets) {
    for (int w = 0; w < 32; ++w) cnt[w * buckets + tid] = static_cast<unsigned short>(cnt[w * buckets + tid] + at);
    for (int i = 0; i < nt; ++i) {
      int* e = items + 1 + 3 * (it - nt + i);
      e[0] = tid < slots ? tid : -1;
      e[1] = at + i * kAdapterItemRows;
      e[2] = min(kAdapterItemRows, n - i * kAdapterItemRows);
    }
  }
  if (tid == kSortThreads - 1) items[0] = it;
  __syncthreads();
  for (int r = lo; r < hi; r += 32) {
    const int row = r + lane;
    int b = -1;
    if (row < hi) { b = ids[row]; if (b < 0 || b >= slots) b = slots; }
    const uint32_t same = __match_any_sync(0xffffffffu, b);
    const int first = b >= 0 ? mine[b] : 0;
    if (b >= 0) order[first + __popc(same & ((1u << lane) - 1))] = row;
    __syncwarp();
    if (b >= 0 && lane == __ffs(same) - 1) mine[b] = static_cast<unsigned short>(first + __popc(same));
    __syncwarp();
  }
}

}  // namespace cb

// Packed by ops/native.py::ADAPTER.
struct CbAdapter {
  const void* x; long long ldx;          // bf16 [rows, k]
  const void* y; long long ldy;          // bf16 [rows, n]
  void* out; long long ldo;              // bf16 [rows, n], may be y
  const void* a;                         // bf16 [slots, sections * rank, k]
  const void* b;                         // bf16 [slots, n, rank]
  const float* scale;                    // [slots]
  const int* ranks;                      // [slots] ranks in use, or null: all
  const int* order; const int* items;    // adapter_rows_kernel's
  void* hi; void* lo;                    // bf16 [rows, sections * rank]: h as a sum of two
  int rows, slots, k, n, rank, sections;
  int width[4];                          // columns of the sections
};

namespace cb {

__device__ __forceinline__ uint4 ldg16(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// h is kept as two bf16: the leading 8 bits of its mantissa cut off, and what is left, rounded: 2^-16 of the value, where one bf16 would
// add 2^-9 to every product.  A value that is not finite is all in the first.
__device__ __forceinline__ void split_h(float v, __nv_bfloat16& hi, __nv_bfloat16& lo) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    hi = __float2bfloat16(v);
    lo = __float2bfloat16(0.f);
    return;
  }
  hi = __ushort_as_bfloat16(static_cast<unsigned short>(u >> 16));
  lo = __float2bfloat16(v - __uint_as_float(u & 0xffff0000u));
}

// h of one item, one section and sixteen rows at a time: the eight warps take turns of 64 along k, the CTAs of a cluster a share of it each; sums are
// joined in their order.  The order of k inside a product is free: a lane's 16 bytes of x and of A are its operands of two products as they lie.
template <int R16>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_down_kernel(const CbAdapter p, int splits) {
  constexpr int R = R16 * 16, NT = R16 * 2;
  extern __shared__ float sh[];                                       // [8][16][R], then the cluster's part [16][R]
  float* part = sh + 8 * 16 * R;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rank_in = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0, team = blockIdx.x / splits, teams = gridDim.x / splits;
  pdl_launch_dependents();
  pdl_wait();
  const int count = p.items[0], units = count * p.sections;
  const int chunk = (((p.k + 63) / 64 + splits - 1) / splits) * 64, k0 = rank_in * chunk, k1 = min(p.k, k0 + chunk);
  const int rt = p.sections * R;
  for (int u = team; u < units; u += teams) {
    const int item = u / p.sections, sec = u - item * p.sections;
    const int slot = p.items[1 + 3 * item], first = p.items[2 + 3 * item], rows = p.items[3 + 3 * item];
    if (slot < 0) continue;
    const float scale = p.scale[slot];
    const int used = p.ranks ? min(R, max(0, p.ranks[slot])) : R;
    const __nv_bfloat16* A = static_cast<const __nv_bfloat16*>(p.a) + (static_cast<size_t>(slot) * rt + sec * R) * p.k;
    for (int m0 = 0; m0 < rows; m0 += 16) {
      const bool in0 = m0 + g < rows, in1 = m0 + g + 8 < rows;
      const __nv_bfloat16* x0 = static_cast<const __nv_bfloat16*>(p.x) + (in0 ? p.order[first + m0 + g] * p.ldx : 0);
      const __nv_bfloat16* x1 = static_cast<const __nv_bfloat16*>(p.x) + (in1 ? p.order[first + m0 + g + 8] * p.ldx : 0);
      float acc[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
      for (int kk = k0 + warp * 64; kk < k1; kk += 8 * 64) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = kk + j * 32 + c * 8;
          const bool in = k < k1;
          const uint4 zero = make_uint4(0, 0, 0, 0);
          const uint4 xa = in && in0 ? ldg16(x0 + k) : zero, xb = in && in1 ? ldg16(x1 + k) : zero;
          const uint32_t f0[4] = {xa.x, xb.x, xa.y, xb.y}, f1[4] = {xa.z, xb.z, xa.w, xb.w};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (t * 8 >= used) break;
            const uint4 w = in ? ldg16(A + static_cast<size_t>(t * 8 + g) * p.k + k) : zero;
            mma_bf16(acc[t], f0, w.x, w.y);
            mma_bf16(acc[t], f1, w.z, w.w);
          }
        }
      }
      float* mine = sh + warp * 16 * R;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        *reinterpret_cast<float2*>(mine + g * R + t * 8 + c * 2) = make_float2(acc[t][0], acc[t][1]);
        *reinterpret_cast<float2*>(mine + (g + 8) * R + t * 8 + c * 2) = make_float2(acc[t][2], acc[t][3]);
      }
      __syncthreads();
      auto put = [&](int e, float v) {
        const int r = e / R;
        if (m0 + r >= rows) return;
        __nv_bfloat16 hi, lo;
        split_h(e - r * R < used ? v * scale : 0.f, hi, lo);          // ranks that are not in use may meet what is not finite in x
        const size_t o = static_cast<size_t>(first + m0 + r) * rt + sec * R + (e - r * R);
        static_cast<__nv_bfloat16*>(p.hi)[o] = hi;
        static_cast<__nv_bfloat16*>(p.lo)[o] = lo;
      };
      for (int e = tid; e < 16 * R; e += kAdapterThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += sh[w * 16 * R + e];
        if (splits == 1) put(e, v);
        else part[e] = v;
      }
      if (splits > 1) {
        cluster_sync_all();
        const uint32_t base = smem_u32(part);
        for (int e = rank_in * kAdapterThreads + tid; e < 16 * R; e += splits * kAdapterThreads) {
          float v = 0.f;
          for (int s = 0; s < splits; ++s) v += ld_cluster_f32(cluster_map(base + e * 4, s));
          put(e, v);
        }
        cluster_sync_all();
      } else {
        __syncthreads();
      }
    }
  }
}

// out = y + h B^T of one item and 256 columns, 32 a warp.  The eight columns of a product are chosen so that a lane ends up with eight neighbours
// of a row: y and out are 16 bytes a lane.  B's operands stay in registers for all rows of the item.
template <int R16>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_up_kernel(const CbAdapter p) {
  constexpr int R = R16 * 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int blocks = (p.n + 255) / 256, units = p.items[0] * blocks, rt = p.sections * R;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = u / blocks, col0 = (u - item * blocks) * 256 + warp * 32;
    if (col0 >= p.n) continue;
    const int slot = p.items[1 + 3 * item], first = p.items[2 + 3 * item], rows = p.items[3 + 3 * item];
    const int col = col0 + c * 8;
    const bool in = col < p.n;
    if (slot < 0) {
      if (p.out == p.y) continue;
      for (int r = g; r < rows; r += 8) {
        const size_t row = p.order[first + r];
        if (in) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + col) = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.y) + row * p.ldy + col);
      }
      continue;
    }
    int sec = 0;
    for (int at = p.width[0]; sec + 1 < p.sections && col0 >= at; at += p.width[sec]) ++sec;
    const int used = p.ranks ? min(R, max(0, p.ranks[slot])) : R;
    // product j, column g is column 8 (g / 2) + 2 j + g % 2 of the 32
    uint32_t b[4][R16][2];
    const __nv_bfloat16* B = static_cast<const __nv_bfloat16*>(p.b) + static_cast<size_t>(slot) * p.n * R;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = col0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
      for (int s = 0; s < R16; ++s) {
        const uint2 w = n < p.n && s * 16 < used ? __ldg(reinterpret_cast<const uint2*>(B + static_cast<size_t>(n) * R + s * 16 + c * 4)) : make_uint2(0, 0);
        b[j][s][0] = w.x;
        b[j][s][1] = w.y;
      }
    }
    for (int m0 = 0; m0 < rows; m0 += 16) {
      const int r0 = m0 + g, r1 = r0 + 8;
      const bool in0 = in && r0 < rows, in1 = in && r1 < rows;
      const size_t row0 = r0 < rows ? p.order[first + r0] : 0, row1 = r1 < rows ? p.order[first + r1] : 0;
      uint4 y0 = make_uint4(0, 0, 0, 0), y1 = y0;
      if (in0) y0 = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.y) + row0 * p.ldy + col);
      if (in1) y1 = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.y) + row1 * p.ldy + col);
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      const size_t h0 = static_cast<size_t>(first + min(r0, rows - 1)) * rt + sec * R + c * 4, h1 = static_cast<size_t>(first + min(r1, rows - 1)) * rt + sec * R + c * 4;
#pragma unroll
      for (int s = 0; s < R16; ++s) {
        if (s * 16 >= used) break;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(half ? p.lo : p.hi);
          const uint2 a0 = *reinterpret_cast<const uint2*>(h + h0 + s * 16), a1 = *reinterpret_cast<const uint2*>(h + h1 + s * 16);
          const uint32_t f[4] = {a0.x, a1.x, a0.y, a1.y};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_bf16(acc[j], f, b[j][s][0], b[j][s][1]);
        }
      }
      auto add = [](uint4 v, const float (&f)[4][4], int o) {
        uint32_t* q = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 w = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(q + j));
          q[j] = pack_bf16x2(w.x + f[j][o], w.y + f[j][o + 1]);
        }
        return v;
      };
      if (in0) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row0 * p.ldo + col) = add(y0, acc, 0);
      if (in1) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row1 * p.ldo + col) = add(y1, acc, 2);
    }
  }
}

template <int R16>
static int adapter_launch(const CbAdapter& p, int items, cudaStream_t stream) {
  constexpr int R = R16 * 16;
  constexpr int smem = 9 * 16 * R * sizeof(float);
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (smem > 48 * 1024 && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(adapter_down_kernel<R16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  const int units = items * p.sections;
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= 592 && p.k / (splits * 2) >= 256) splits *= 2;
  const int teams = min(units, 592 / splits);
  e = launch(adapter_down_kernel<R16>, dim3(teams * splits), dim3(kAdapterThreads), smem, stream, dim3(splits, 1, 1), p, splits);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int blocks = (p.n + 255) / 256;
  return static_cast<int>(launch(adapter_up_kernel<R16>, dim3(min(items * blocks, 148 * 4)), dim3(kAdapterThreads), 0, stream, p));
}

static int adapter_items(int rows, int slots) { return rows / kAdapterItemRows + min(slots + 1, rows); }

}  // namespace cb

extern "C" {

// Most work items that `rows` rows over `slots` adapters can make: `items` of cb_adapter_rows holds 1 + 3 times as many.
int cb_adapter_items(int rows, int slots) { return rows <= 0 || slots <= 0 ? 0 : cb::adapter_items(rows, slots); }

int cb_adapter_rows(const void* ids, int rows, int slots, void* order, void* items, void* stream) {
  using namespace cb;
  if (rows < 0 || rows > kAdapterMaxRows || slots < 1 || slots > kAdapterMaxSlots) return -10;
  const int smem = 32 * (slots + 1) * static_cast<int>(sizeof(unsigned short));
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(adapter_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 32 * (kAdapterMaxSlots + 1) * sizeof(unsigned short));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(launch(adapter_rows_kernel, dim3(1), dim3(kSortThreads), smem, static_cast<cudaStream_t>(stream), static_cast<const int*>(ids), rows, slots,
                                 static_cast<int*>(order), static_cast<int*>(items)));
}

int cb_adapter_add(const CbAdapter* p, void* stream) {
  using namespace cb;
  if (p->rows < 0 || p->rows > kAdapterMaxRows || p->slots < 1 || p->slots > kAdapterMaxSlots || p->k < 8 || p->k % 8 || p->n < 8 || p->n % 8) return -10;
  if (p->sections < 1 || p->sections > kAdapterSections || p->ldx % 8 || p->ldy % 8 || p->ldo % 8) return -11;
  int n = 0;
  for (int i = 0; i < p->sections; ++i) {
    if (p->width[i] < 8 || (i + 1 < p->sections && p->width[i] % 32)) return -12;
    n += p->width[i];
  }
  if (n != p->n) return -12;
  if (((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->y) | reinterpret_cast<uintptr_t>(p->out) | reinterpret_cast<uintptr_t>(p->a) | reinterpret_cast<uintptr_t>(p->b) |
        reinterpret_cast<uintptr_t>(p->hi) | reinterpret_cast<uintptr_t>(p->lo)) & 15) != 0)
    return -13;
  if (p->rows == 0) return 0;
  const int items = adapter_items(p->rows, p->slots);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->rank) {
    case 16: return adapter_launch<1>(*p, items, s);
    case 32: return adapter_launch<2>(*p, items, s);
    case 64: return adapter_launch<4>(*p, items, s);
    case 128: return adapter_launch<8>(*p, items, s);
  }
  return -14;
}

}  // extern "C"
