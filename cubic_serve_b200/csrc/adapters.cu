// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + scale[s] (x[t] A[s]^T) B[s]^T,  s = adapter of row t (none: out[t] = y[t]).
// A projection made of sections (q | k | v, gate | up) has an A of its own for each: A[s] stacks them, and the columns of section j see
// ranks [j rank, (j + 1) rank).
//
// `adapter_rows_kernel` sorts a step's rows by adapter, once for all projections of all layers.  Up to 512 rows `adapter_few_kernel` makes
// h = scale x A^T of up to sixteen rows of an adapter and adds h B^T, in one launch.  From there on `adapter_down_tile_kernel` makes h of up to 64 rows and
// `adapter_up_kernel` adds h B^T to strips of sixteen.
//
// Bound by memory: with few rows by A and B of the adapters in use, with many by y and out.  The products run on
// mma.sync m16n8k16 with operands that go from global memory to registers: rank 16 makes 16 products of every byte of x, far from
// what would keep tensor memory busy.
#include "ptx.cuh"
#include "mma.cuh"
#include "launch.cuh"

namespace cb {

// Up to here a work item is sixteen rows and A is streamed through registers, from here on it is 64 and A and x come by tiles.  A layer of rank 16, by tiles and
// by sixteens: 331 rows over 2 adapters 82 and 57 us; 640 over 2, 16 and 64 76, 86, 112 and 82, 87, 128; 1024 98, 103, 122 and 90, 93, 147; 2048 143, 153, 184 and 151, 154, 251.
// 640 rows of rank 32 89, 98, 130 and 95, 100, 154; of 64 130, 138, 206 and 133, 139, 230; of 128 176, 208, 354 and 219, 229, 398.  1024 rows of rank 32 112, 117, 140 and 102, 106, 171;
// of 64 162, 174, 215 and 138, 145, 248; of 128 227, 265, 364 and 223, 237, 431: with few adapters the sixteens are ahead beyond the limit, with many they are not.
static constexpr int kAdapterFewRows = 512;
static constexpr int adapter_item_rows(int rows) { return rows <= kAdapterFewRows ? 16 : 64; }
static constexpr int kAdapterMaxSlots = 1023;
static constexpr int kAdapterMaxRows = 65535;
static constexpr int kAdapterSections = 4;
static constexpr long long kAdapterMaxStride = 1 << 30;               // in bytes a row fits in 32 bits
static constexpr int kSortThreads = 1024;
static constexpr int kAdapterThreads = 256;

// ------------------------------------------------------------------ rows by adapter
// order[]: the step's rows by adapter, a row's place among its adapter's by its index; rows without one last.
// items[]: [0] = count, then {adapter (-1: none), first place, rows} of up to 16 or 64 rows.
// strips[]: [0] = count, from [4] on {adapter, first place, rows, 0} of up to 16.
// One CTA: a warp counts the adapters of its share of the rows, the counts become places, a second look at the ids fills them.  8192 rows
// are two rounds of 8 steps a warp.
__global__ void __launch_bounds__(kSortThreads)
adapter_rows_kernel(const int* ids, int rows, int slots, int* order, int* items, int* strips) {
  extern __shared__ unsigned short cnt[];                             // [warps][buckets]
  __shared__ int warp_sum[3][32], base[3][kAdapterMaxSlots + 2];      // rows, items and strips of the buckets before
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, buckets = slots + 1;
  const int share = (((rows + 31) >> 5) + 31) & ~31, lo = min(rows, warp * share), hi = min(rows, lo + share);
  const int warps = rows ? (rows + share - 1) / share : 0;            // that have any rows
  for (int i = tid; i < warps * buckets; i += kSortThreads) cnt[i] = 0;
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
  // counts of the warps before, then of the buckets before
  int n = 0;
  if (tid < buckets) {
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int c = cnt[w * buckets + tid];
      cnt[w * buckets + tid] = static_cast<unsigned short>(n);
      n += c;
    }
  }
  const int per = adapter_item_rows(rows);
  int sum[3] = {n, (n + per - 1) / per, (n + 15) / 16};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int a = __shfl_up_sync(0xffffffffu, sum[i], o);
      if (lane >= o) sum[i] += a;
    }
  if (lane == 31) for (int i = 0; i < 3; ++i) warp_sum[i][warp] = sum[i];
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      int v = warp_sum[i][lane];
      const int own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += a;
      }
      warp_sum[i][lane] = v - own;
    }
  }
  if (tid == 0) base[0][0] = base[1][0] = base[2][0] = 0;
  __syncthreads();
  if (tid < buckets) {
#pragma unroll
    for (int i = 0; i < 3; ++i) base[i][tid + 1] = sum[i] + warp_sum[i][warp];
    const int at = base[0][tid + 1] - n;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) cnt[w * buckets + tid] = static_cast<unsigned short>(cnt[w * buckets + tid] + at);
  }
  __syncthreads();
  // both lists, an entry a thread
  auto bucket_of = [&](const int* upto, int e) {                      // the last that starts at or before e
    int a = 0, b = buckets;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (upto[mid] <= e) a = mid; else b = mid;
    }
    return a;
  };
  for (int e = tid; e < base[1][buckets]; e += kSortThreads) {
    const int b = bucket_of(base[1], e), off = (e - base[1][b]) * per;
    items[1 + 3 * e] = b < slots ? b : -1;
    items[2 + 3 * e] = base[0][b] + off;
    items[3 + 3 * e] = min(per, base[0][b + 1] - base[0][b] - off);
  }
  for (int e = tid; e < base[2][buckets]; e += kSortThreads) {
    const int b = bucket_of(base[2], e), off = (e - base[2][b]) * 16;
    reinterpret_cast<int4*>(strips)[1 + e] = make_int4(b < slots ? b : -1, base[0][b] + off, min(16, base[0][b + 1] - base[0][b] - off), 0);
  }
  if (tid == 0) { items[0] = base[1][buckets]; strips[0] = base[2][buckets]; }
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
  const void* a;                         // bf16 [slots, ceil(k / 32), sections * rank, 32]: what is read together lies together
  const void* b;                         // bf16 [slots, n, rank]
  const float* scale;                    // [slots]
  const int* ranks;                      // [slots] ranks in use by any section
  const uint32_t* section_ranks;         // [slots] ranks in use, a byte a section; B is zero behind them
  const int* order; const int* items; const int* strips;         // adapter_rows_kernel's
  void* hi; void* lo;                    // bf16 [rows, sections * rank]: h as a sum of two
  int rows, slots, k, n, rank, sections;
  int width[4];                          // columns of the sections
};

namespace cb {

// A section has ranks of its own (none, if the adapter leaves it as it is): an infinity in x makes NaN of the zeros behind them, and that must meet no column.
__device__ __forceinline__ int ranks_in(uint32_t section_ranks, int section) { return static_cast<int>(section_ranks >> 8 * section & 0xffu); }
__device__ __forceinline__ int most_ranks(uint32_t section_ranks) {
  const uint32_t two = __vmaxu4(section_ranks, section_ranks >> 16);
  return static_cast<int>(max(two & 0xffu, two >> 8 & 0xffu));
}

// For A and B alone: what another kernel of the stream writes may change after this one has started, which the read-only path does not allow.
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

// What is left to do with a sum: scale it, and write its two parts.
__device__ __forceinline__ void put_h(const CbAdapter& p, float v, float scale, bool in_use, size_t at) {
  __nv_bfloat16 hi, lo;
  split_h(in_use ? v * scale : 0.f, hi, lo);                          // ranks that are not in use may meet what is not finite in x
  static_cast<__nv_bfloat16*>(p.hi)[at] = hi;
  static_cast<__nv_bfloat16*>(p.lo)[at] = lo;
}

// Few rows: both products of an item of up to sixteen rows by a cluster, in one launch.  The CTAs have a share of k each, make their part of h for all sections,
// add the parts up from one another's shared memory, tell all of them the sums, and go on with a share of the columns each.
//
// First product: A is the operand of sixteen, rows of x those of eight, for most adapters of a decode step have no more.  The eight warps of all CTAs take turns
// of 32 along k.  The order of k inside a product is free: a lane's 16 bytes of x and of A are its operands of two products as they lie.  64 ranks
// at a time, one turn of a warp on its way while another is multiplied.
// Second product: as in adapter_up_kernel, with h from shared memory and sixteen rows at most.
//
// A layer's four projections (4096 -> 6144 of three sections, 4096 -> 4096, 4096 -> 24576 of two, 12288 -> 4096) one after the other: one row of rank 16 takes
// 27 us (a launch's start, two waits for the cluster and four trips to memory, 6.7 us each), 48 rows, 36 of them over nine adapters of rank 32, 46 us, 256 rows, 240 over 60 of rank
// 64 133 us (634 MB: 4.8 TB/s; with a launch for each product 27, 50 and 150).
template <int R16, int MT>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_few_kernel(const CbAdapter p, int splits) {
  constexpr int R = R16 * 16, RP = 68, W = 16 * MT;
  extern __shared__ __align__(16) unsigned char few[];
  const int rt = p.sections * R, tiles = rt / 16, hp = rt + 8;        // row pitch of h
  float* red = reinterpret_cast<float*>(few);                         // [8 warps][16 rows][RP]
  float* part = red + 8 * 16 * RP;                                    // [16][rt]
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(part + 16 * rt);                  // [2 parts][16][hp]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rank_in = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0, team = blockIdx.x / splits, teams = gridDim.x / splits;
  pdl_launch_dependents();
  pdl_wait();
  const int4* list = reinterpret_cast<const int4*>(p.strips) + 1;     // adapter, first place, rows
  const int items = p.strips[0], turns = (p.k + 31) >> 5, step = 8 * splits, n = p.n;
  const bool in_place = p.out == p.y;
  int4 next = list[team];                                             // on its way with their number
  for (int item = team; item < items; item += teams) {
    const int slot = next.x, first = next.y, rows = next.z;
    if (item + teams < items) next = list[item + teams];
    if (slot < 0) {                                                   // rows without an adapter
      if (in_place) continue;
      const int chunks = n / 8;
      for (int e = rank_in * kAdapterThreads + tid; e < rows * chunks; e += splits * kAdapterThreads) {
        const size_t row = p.order[first + e / chunks];
        const int col = e % chunks * 8;
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + col) = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.y) + row * p.ldy + col);
      }
      continue;
    }
    const uint32_t used = p.section_ranks[slot];
    const float scale = p.scale[slot];
    const bool in0 = g < rows, in1 = g + 8 < rows, both = rows > 8;
    const __nv_bfloat16* x0 = static_cast<const __nv_bfloat16*>(p.x) + (in0 ? p.order[first + g] * p.ldx : 0) + c * 8;
    const __nv_bfloat16* x1 = static_cast<const __nv_bfloat16*>(p.x) + (in1 ? p.order[first + g + 8] * p.ldx : 0) + c * 8;
    for (int q0 = 0; q0 < tiles; q0 += 4) {
      const __nv_bfloat16* A = static_cast<const __nv_bfloat16*>(p.a) + (static_cast<size_t>(slot) * turns * rt + q0 * 16) * 32 + lane * 8;
      bool on[4];                                                     // tiles of sixteen that hold ranks in use
#pragma unroll
      for (int t = 0; t < 4; ++t) on[t] = q0 + t < tiles && (R16 == 1 ? used != 0 : (q0 + t) % R16 * 16 < ranks_in(used, (q0 + t) / R16));
      float acc[4][2][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[t][h][0] = acc[t][h][1] = acc[t][h][2] = acc[t][h][3] = 0.f;
      uint4 w[2][4][2], xa[2], xb[2];
      auto load = [&](int b, int at) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const bool in = at < turns, in_x = at * 32 + c * 8 < p.k;
        xa[b] = in_x && in0 ? *reinterpret_cast<const uint4*>(x0 + at * 32) : zero;
        xb[b] = in_x && in1 ? *reinterpret_cast<const uint4*>(x1 + at * 32) : zero;
        const __nv_bfloat16* from = A + static_cast<size_t>(at) * rt * 32;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) w[b][t][h] = in && on[t] ? ldg16(from + (t * 16 + h * 8) * 32) : zero;
      };
      auto multiply = [&](int b) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint4 &lo = w[b][t][0], &hi = w[b][t][1];
          const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
          mma_bf16(acc[t][0], f0, xa[b].x, xa[b].y);
          mma_bf16(acc[t][0], f1, xa[b].z, xa[b].w);
          if (both) {
            mma_bf16(acc[t][1], f0, xb[b].x, xb[b].y);
            mma_bf16(acc[t][1], f1, xb[b].z, xb[b].w);
          }
        }
      };
      const int t0 = rank_in * 8 + warp;
      load(0, t0);
      for (int t = t0; t < turns; t += 2 * step) {
        load(1, t + step);
        multiply(0);
        load(0, t + 2 * step);
        multiply(1);
      }
      float* mine = red + warp * 16 * RP;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h && !both) break;
          float* at = mine + (h * 8 + c * 2) * RP + t * 16 + g;
          at[0] = acc[t][h][0];
          at[RP] = acc[t][h][1];
          at[8] = acc[t][h][2];
          at[RP + 8] = acc[t][h][3];
        }
      __syncthreads();
      const int width = min(64, rt - q0 * 16);
      for (int e = tid; e < rows * 64; e += kAdapterThreads) {
        const int r = e >> 6, k = e & 63;
        if (k >= width) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += red[(q * 16 + r) * RP + k];
        part[r * rt + q0 * 16 + k] = v;
      }
      __syncthreads();
    }
    // B and y of the warp's first columns come while the sums are exchanged
    int row[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i) row[e][i] = e * 8 + 2 * c + i < rows ? p.order[first + e * 8 + 2 * c + i] : -1;
    // product t, places g and g + 8: columns 2 t and 2 t + 1 of the lane's
    uint32_t b[MT][R16][4], y[2][2][MT];
    auto load_columns = [&](int u) {
      const int col = u * W + g * 2 * MT;
      const bool in = col < n;
      const int most = most_ranks(used);
      const __nv_bfloat16* B = static_cast<const __nv_bfloat16*>(p.b) + (static_cast<size_t>(slot) * n + col) * R;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const __nv_bfloat16* at = B + (2 * t + k) * R;
          if (R16 == 1) {
            const uint2 v = in && used ? __ldg(reinterpret_cast<const uint2*>(at + c * 4)) : make_uint2(0, 0);
            b[t][0][k] = v.x;
            b[t][0][2 + k] = v.y;
          } else {
#pragma unroll
            for (int s = 0; s < R16 / 2; ++s) {
              const uint4 v = in && s * 32 < most ? ldg16(at + s * 32 + c * 8) : make_uint4(0, 0, 0, 0);
              b[t][2 * s][k] = v.x;
              b[t][2 * s][2 + k] = v.y;
              b[t][2 * s + 1][k] = v.z;
              b[t][2 * s + 1][2 + k] = v.w;
            }
          }
        }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int t = 0; t < MT; ++t) y[e][i][t] = 0;
          if (!in || row[e][i] < 0) continue;
          const __nv_bfloat16* at = static_cast<const __nv_bfloat16*>(p.y) + row[e][i] * p.ldy + col;
          if (MT == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            y[e][i][0] = v.x; y[e][i][1] = v.y; y[e][i][MT - 2] = v.z; y[e][i][MT - 1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            y[e][i][0] = v.x; y[e][i][1] = v.y;
          }
        }
    };
    load_columns(rank_in * 8 + warp);
    // two ranks a thread: the sum over the CTAs in their order, and its two parts to all of them
    if (splits > 1) cluster_sync_all();
    const uint32_t part_at = smem_u32(part), hs_at = smem_u32(hs);
    for (int e = rank_in * kAdapterThreads + tid; e < 8 * rt; e += splits * kAdapterThreads) {
      const int r = e / (rt / 2), k = e % (rt / 2) * 2;
      float v[2] = {0.f, 0.f};
      if (r < rows) {
        if (splits > 1) {
          float2 q[8];
#pragma unroll
          for (int s = 0; s < 8; ++s) {
            q[s] = make_float2(0.f, 0.f);
            if (s < splits) {
              asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(q[s].x), "=f"(q[s].y) : "r"(cluster_map(part_at + (r * rt + k) * 4, s)) : "memory");
            }
          }
#pragma unroll
          for (int s = 0; s < 8; ++s) { v[0] += q[s].x; v[1] += q[s].y; }
        } else {
          v[0] = part[r * rt + k];
          v[1] = part[r * rt + k + 1];
        }
      }
      uint32_t hi = 0, lo = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __nv_bfloat16 a, b;
        split_h((k + i) % R < ranks_in(used, (k + i) / R) ? v[i] * scale : 0.f, a, b);       // ranks that are not in use may have met what is not finite in x
        hi |= static_cast<uint32_t>(__bfloat16_as_ushort(a)) << 16 * i;
        lo |= static_cast<uint32_t>(__bfloat16_as_ushort(b)) << 16 * i;
      }
      const uint32_t to = hs_at + (r * hp + k) * 2;
      if (splits > 1) {
        for (int s = 0; s < splits; ++s) {
          st_cluster_u32(cluster_map(to, s), hi);
          st_cluster_u32(cluster_map(to + 16 * hp * 2, s), lo);
        }
      } else {
        *reinterpret_cast<uint32_t*>(hs + r * hp + k) = hi;
        *reinterpret_cast<uint32_t*>(hs + (16 + r) * hp + k) = lo;
      }
    }
    if (splits > 1) cluster_sync_all(); else __syncthreads();
    for (int u = rank_in * 8 + warp; u * W < n; u += step) {
      const int col0 = u * W, col = col0 + g * 2 * MT;
      const bool in = col < n;
      int sec = 0;
      for (int at = p.width[0]; sec + 1 < p.sections && col0 >= at; at += p.width[sec]) ++sec;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e * 8 >= rows) break;
        float acc[MT][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            acc[t][i] = __uint_as_float(y[e][i][t] << 16);
            acc[t][2 + i] = __uint_as_float(y[e][i][t] & 0xffff0000u);
          }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const __nv_bfloat16* h = hs + (half * 16 + e * 8 + g) * hp + sec * R;
          if (R16 == 1) {
            const uint2 v = *reinterpret_cast<const uint2*>(h + c * 4);
#pragma unroll
            for (int t = 0; t < MT; ++t) mma_bf16(acc[t], b[t][0], v.x, v.y);
          } else {
#pragma unroll
            for (int s = 0; s < R16 / 2; ++s) {
              const uint4 v = *reinterpret_cast<const uint4*>(h + s * 32 + c * 8);
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                mma_bf16(acc[t], b[t][2 * s], v.x, v.y);
                mma_bf16(acc[t], b[t][2 * s + 1], v.z, v.w);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!in || row[e][i] < 0) continue;
          __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.out) + row[e][i] * p.ldo + col;
          if (MT == 4) {
            *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(acc[0][i], acc[0][2 + i]), pack_bf16x2(acc[1][i], acc[1][2 + i]),
                                                       pack_bf16x2(acc[MT - 2][i], acc[MT - 2][2 + i]), pack_bf16x2(acc[MT - 1][i], acc[MT - 1][2 + i]));
          } else {
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[0][i], acc[0][2 + i]), pack_bf16x2(acc[1][i], acc[1][2 + i]));
          }
        }
      }
      if ((u + step) * W < n) load_columns(u + step);
    }
    if (splits == 1) __syncthreads();                                 // h is read until here
  }
}

// h of many rows: a CTA makes 64 rows x (16 NT) ranks, whatever sections these belong to, so that x is read once; stages of 64 H along k come by asynchronous
// copies.  Four warps by two: 16 rows and half of the ranks each.  The CTAs of a cluster have a share of k each.
// 8192 rows of rank 16, a layer: 127 us for 402 MB of x (3.2 TB/s) and as much again of A out of L2 at 64 rows a tile; two more stages in flight change nothing.
template <int NT>
struct DownTile {
  static constexpr int NR = NT * 16, H = NT <= 4 ? 2 : 1, kStages = NT <= 4 ? 3 : 4;
  static constexpr int kHalfBytes = (64 + NR) * 128, kStageBytes = H * kHalfBytes, kBytes = kStages * kStageBytes, SP = NR + 2;
};
template <int NT>
__global__ void __launch_bounds__(kAdapterThreads, 2)
adapter_down_tile_kernel(const CbAdapter p, int splits) {
  using T = DownTile<NT>;
  constexpr int NR = T::NR, H = T::H, kStages = T::kStages, SP = T::SP, AR = (NR + 31) / 32;
  extern __shared__ __align__(128) unsigned char st[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp & 3, wn = warp >> 2;
  const int rank_in = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0, team = blockIdx.x / splits, teams = gridDim.x / splits;
  pdl_launch_dependents();
  pdl_wait();
  const int rt = p.sections * p.rank, parts = (rt + NR - 1) / NR, units = p.items[0] * parts, stages = (p.k + 64 * H - 1) / (64 * H);
  const int turns = (p.k + 31) >> 5, share = (stages + splits - 1) / splits, s0 = rank_in * share, s1 = min(stages, s0 + share);
  const uint32_t base = smem_u32(st);
  for (int u = team; u < units; u += teams) {
    const int item = u / parts, r0 = (u - item * parts) * NR;
    const int slot = p.items[1 + 3 * item], first = p.items[2 + 3 * item], rows = p.items[3 + 3 * item];
    if (slot < 0) continue;
    const int used = min(p.rank, max(0, p.ranks[slot]));
    const int row = tid >> 3, ch = tid & 7;                           // a thread's 16 bytes of rows row, row + 32, ...
    const __nv_bfloat16 *xr[2], *ar[AR];
    bool xin[2], ain[AR];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xin[i] = row + 32 * i < rows;
      xr[i] = static_cast<const __nv_bfloat16*>(p.x) + (xin[i] ? p.order[first + row + 32 * i] * p.ldx : 0) + ch * 8;
    }
#pragma unroll
    for (int i = 0; i < AR; ++i) {
      const int r = r0 + row + 32 * i;
      ain[i] = row + 32 * i < NR && r < rt && r % p.rank < used;
      ar[i] = static_cast<const __nv_bfloat16*>(p.a) + ((static_cast<size_t>(slot) * turns + ch / 4) * rt + (ain[i] ? r : 0)) * 32 + ch % 4 * 8;
    }
    const uint32_t to0 = base + row * 128 + ((ch ^ (row & 7)) << 4);
    auto fetch = [&](int s, int buf) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int k = (s * H + h) * 64;
        const bool in = s < s1 && k + ch * 8 < p.k;
        const uint32_t to = to0 + buf * T::kStageBytes + h * T::kHalfBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) cp_async16(to + i * 32 * 128, in && xin[i] ? xr[i] + k : p.x, in && xin[i]);
#pragma unroll
        for (int i = 0; i < AR; ++i)
          if (row + 32 * i < NR) cp_async16(to + (64 + i * 32) * 128, in && ain[i] ? static_cast<const void*>(ar[i] + static_cast<size_t>(k) * rt) : p.a, in && ain[i]);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(s0 + i, i);
    int buf = 0;
    for (int s = s0; s < s1; ++s) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncthreads();
      fetch(s + kStages - 1, (buf + kStages - 1) % kStages);
      if (wm * 16 < rows) {
#pragma unroll
        for (int kk = 0; kk < 4 * H; ++kk) {
          const uint32_t xs = base + buf * T::kStageBytes + (kk / 4) * T::kHalfBytes, as = xs + 64 * 128;
          const int k = kk & 3;
          uint32_t a[4];
          const int r = wm * 16 + (lane & 15), kc = k * 2 + (lane >> 4);
          ldsm4(a, xs + r * 128 + ((kc ^ (r & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; t += 2) {
            uint32_t b[4];
            const int n = (wn * NT + t) * 8 + (lane & 7) + (t + 1 < NT ? (lane >> 4) * 8 : 0), bc = k * 2 + (lane >> 3 & 1);
            ldsm4(b, as + n * 128 + ((bc ^ (n & 7)) << 4));
            mma_bf16(acc[t], a, b[0], b[1]);
            if (t + 1 < NT) mma_bf16(acc[t + 1], a, b[2], b[3]);
          }
        }
      }
      buf = (buf + 1) % kStages;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    const float scale = p.scale[slot];
    const uint32_t by_section = p.section_ranks[slot];
    float* part = reinterpret_cast<float*>(st);                       // [64][SP]
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* at = part + (wm * 16 + (lane >> 2)) * SP + (wn * NT + t) * 8 + (lane & 3) * 2;
      *reinterpret_cast<float2*>(at) = make_float2(acc[t][0], acc[t][1]);
      *reinterpret_cast<float2*>(at + 8 * SP) = make_float2(acc[t][2], acc[t][3]);
    }
    if (splits > 1) cluster_sync_all(); else __syncthreads();
    const int width = min(NR, rt - r0);
    for (int e = rank_in * kAdapterThreads + tid; e < rows * NR; e += splits * kAdapterThreads) {
      const int r = e / NR, k = e % NR;
      if (k >= width) continue;
      float v = 0.f;
      if (splits > 1) {
        float q[8];
        const uint32_t at = smem_u32(part + r * SP + k);
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s] = s < splits ? ld_cluster_f32(cluster_map(at, s)) : 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) v += q[s];
      } else {
        v = part[r * SP + k];
      }
      put_h(p, v, scale, (r0 + k) % p.rank < ranks_in(by_section, (r0 + k) / p.rank), static_cast<size_t>(first + r) * rt + r0 + k);
    }
    if (splits > 1) cluster_sync_all(); else __syncthreads();
  }
}

// out = y + h B^T of strips of sixteen rows, 16 MT columns a warp.  B is the operand of sixteen, rows of h those of eight.  Which columns a product has is
// free: they are chosen so that a lane ends up with 2 MT neighbours of two rows, and eight lanes with a row of 16 MT.  A warp keeps its columns for a run of
// strips and B's operands in registers as long as these are of one adapter; the products add to y, which is rounded once.  y comes through a ring of the
// warp's own, three strips ahead, and goes back through it: eight lanes copy a line of y, and a line of out.  (A lane's own columns straight from global
// memory were four lines a quarter of a warp: 71 % of the load and store unit's cycles.)
// 8192 rows of rank 16, 24576 columns: 160 us for 805 MB of y and out (5.0 TB/s); a bare copy in the same pattern takes 133 to 143.
template <int R16, int MT>
__global__ void __launch_bounds__(kAdapterThreads, R16 * MT <= 4 ? 3 : 2)
adapter_up_kernel(const CbAdapter p) {
  constexpr int R = R16 * 16, W = 16 * MT, kRing = 4, CH = 2 * MT, RP = 32 / CH, I = 16 / RP;     // 16-byte chunks of a row, rows of a copy, copies
  constexpr bool AHEAD = R16 <= 2;                                             // registers for the next strip's h
  extern __shared__ __align__(16) unsigned char ring[];                        // [8 warps][kRing][16 rows][CH chunks]
  __shared__ int ring_row[8][kRing][16];                                       // which rows they are
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3, rr = lane / CH, rc = lane % CH;
  unsigned char* mine = ring + warp * kRing * 256 * CH;
  const uint32_t mine_at = smem_u32(mine);
  // rows of eight fall on all banks: MT 4 by their number, MT 2 (64 bytes a row) by that of their pair
  auto place = [](int row, int chunk) { return static_cast<uint32_t>((row * CH + (chunk ^ (MT == 4 ? row & 7 : row >> 1 & 3))) * 16); };
  uint32_t own[2], copy[I > 1 ? 2 : 1];                                        // places of the lane: its products' rows 2 c + i, the rows it copies; the next eight 128 CH on
#pragma unroll
  for (int i = 0; i < 2; ++i) own[i] = MT == 4 ? place(2 * c + i, g) : place(2 * c + i, g >> 1) + (g & 1) * 8;
#pragma unroll
  for (int i = 0; i < 8 / RP; ++i) copy[i] = place(rr + i * RP, rc);
  auto copy_at = [&](int i) { return copy[i % (8 / RP)] + i / (8 / RP) * 128 * CH; };
  pdl_launch_dependents();
  pdl_wait();
  const int n = p.n, blocks = (n + W - 1) / W, strips = p.strips[0], rt = p.sections * R, warps = gridDim.x * 8;
  const int runs = min(strips, max(1, warps / blocks)), tasks = runs * blocks;         // runs of strips, of about the same length
  const uint32_t ldy = static_cast<uint32_t>(p.ldy) * 2, ldo = static_cast<uint32_t>(p.ldo) * 2;
  const bool in_place = p.out == p.y;
  const int4* list = reinterpret_cast<const int4*>(p.strips) + 1;              // adapter, first place, rows
  const ptrdiff_t lo_off = static_cast<const __nv_bfloat16*>(p.lo) - static_cast<const __nv_bfloat16*>(p.hi);
  for (int task = blockIdx.x * 8 + warp; task < tasks; task += warps) {
    const int run = task / blocks, col0 = (task - run * blocks) * W, col = col0 + g * 2 * MT;
    const int s0 = static_cast<int>(static_cast<long long>(strips) * run / runs), s1 = static_cast<int>(static_cast<long long>(strips) * (run + 1) / runs);
    const bool in = col < n, in_copy = col0 + rc * 8 < n;
    int sec = 0;
    for (int at = p.width[0]; sec + 1 < p.sections && col0 >= at; at += p.width[sec]) ++sec;
    const char* from = static_cast<const char*>(p.y) + (col0 + rc * 8) * 2;
    char* to = static_cast<char*>(p.out) + (col0 + rc * 8) * 2;
    const __nv_bfloat16* h0 = static_cast<const __nv_bfloat16*>(p.hi) + static_cast<size_t>(g) * rt + sec * R + c * (R16 == 1 ? 4 : 8);
    // what is fetched next: its strip and rows (one a lane) are looked up a step before
    int f = s0, put = 0, get = 0, ahead = 0;
    int4 f_strip = make_int4(-1, 0, 0, 0);
    auto look_up = [&]() {
      if (f >= s1) return;
      f_strip = list[f];
      if (lane < f_strip.z) ahead = p.order[f_strip.y + lane];
    };
    auto fetch = [&]() {
      if (f < s1) {
        const bool skip = in_place && f_strip.x < 0;
        if (lane < 16) ring_row[warp][put][lane] = ahead;
        const int left = in_copy && !skip ? f_strip.z - rr : 0;
#pragma unroll
        for (int i = 0; i < I; ++i)
          cp_async16(mine_at + put * 256 * CH + copy_at(i), from + static_cast<size_t>(ldy) * static_cast<uint32_t>(__shfl_sync(0xffffffffu, ahead, rr + i * RP)), i * RP < left);
        ++f;
        look_up();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      put = (put + 1) % kRing;
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < kRing - 1; ++i) fetch();
    uint2 h[AHEAD ? 2 : 1][2][R16];                                            // of eight rows, both parts
    // rows behind the strip's last are another's, or the spare ones behind the buffer's: what comes of them is not written
    auto load_h = [&](int e_, int first) {
      const int e = AHEAD ? e_ : 0;
      const __nv_bfloat16* at = h0 + static_cast<size_t>(first + e_ * 8) * rt;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (R16 == 1) {
          h[e][half][0] = *reinterpret_cast<const uint2*>(at + (half ? lo_off : 0));
        } else {
#pragma unroll
          for (int s = 0; s < R16 / 2; ++s) {
            const uint4 v = *reinterpret_cast<const uint4*>(at + (half ? lo_off : 0) + s * 32);
            h[e][half][2 * s] = make_uint2(v.x, v.y);
            h[e][half][2 * s + 1] = make_uint2(v.z, v.w);
          }
        }
      }
    };
    int4 strip = list[s0];
    if (AHEAD) { load_h(0, strip.y); load_h(1, strip.y); }
    uint32_t b[MT][R16][4];
    int held = -2, used = 0;                                                   // the adapter whose B is in registers
#pragma unroll 1
    for (int s = s0; s < s1; ++s) {
      if (strip.x != held) {
        held = strip.x;
        used = held < 0 ? 0 : min(R, max(0, p.ranks[held]));
        // product t, places g and g + 8: columns 2 t and 2 t + 1 of the lane's
        const __nv_bfloat16* B = static_cast<const __nv_bfloat16*>(p.b) + (static_cast<size_t>(max(held, 0)) * n + col) * R;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const __nv_bfloat16* at = B + (2 * t + k) * R;
            if (R16 == 1) {
              const uint2 v = in && used ? __ldg(reinterpret_cast<const uint2*>(at + c * 4)) : make_uint2(0, 0);
              b[t][0][k] = v.x;
              b[t][0][2 + k] = v.y;
            } else {
#pragma unroll
              for (int q = 0; q < R16 / 2; ++q) {
                const uint4 v = in && q * 32 < used ? ldg16(at + q * 32 + c * 8) : make_uint4(0, 0, 0, 0);
                b[t][2 * q][k] = v.x;
                b[t][2 * q][2 + k] = v.y;
                b[t][2 * q + 1][k] = v.z;
                b[t][2 * q + 1][2 + k] = v.w;
              }
            }
          }
      }
      const int first = strip.y, left = in_copy && !(in_place && held < 0) ? strip.z - rr : 0, rows = strip.z;
      if (s + 1 < s1) strip = list[s + 1];
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      __syncwarp();
      unsigned char* slot = mine + get * 256 * CH;
      if (used) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (R16 > 1 && e * 8 >= rows) break;
          if (!AHEAD) load_h(e, first);
          float acc[MT][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned char* at = slot + own[i] + e * 128 * CH;
            uint32_t y[MT];
            if (MT == 4) {
              const uint4 v = *reinterpret_cast<const uint4*>(at);
              y[0] = v.x; y[1] = v.y; y[MT - 2] = v.z; y[MT - 1] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(at);
              y[0] = v.x; y[1] = v.y;
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              acc[t][i] = __uint_as_float(y[t] << 16);
              acc[t][2 + i] = __uint_as_float(y[t] & 0xffff0000u);
            }
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int k = 0; k < R16; ++k)
#pragma unroll
              for (int t = 0; t < MT; ++t) mma_bf16(acc[t], b[t][k], h[AHEAD ? e : 0][half][k].x, h[AHEAD ? e : 0][half][k].y);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            unsigned char* at = slot + own[i] + e * 128 * CH;
            if (MT == 4) {
              *reinterpret_cast<uint4*>(at) = make_uint4(pack_bf16x2(acc[0][i], acc[0][2 + i]), pack_bf16x2(acc[1][i], acc[1][2 + i]),
                                                         pack_bf16x2(acc[MT - 2][i], acc[MT - 2][2 + i]), pack_bf16x2(acc[MT - 1][i], acc[MT - 1][2 + i]));
            } else {
              *reinterpret_cast<uint2*>(at) = make_uint2(pack_bf16x2(acc[0][i], acc[0][2 + i]), pack_bf16x2(acc[1][i], acc[1][2 + i]));
            }
          }
        }
        __syncwarp();
      }
      if (AHEAD && s + 1 < s1) { load_h(0, strip.y); load_h(1, strip.y); }
#pragma unroll
      for (int i = 0; i < I; ++i)
        if (i * RP < left)
          *reinterpret_cast<uint4*>(to + static_cast<size_t>(ldo) * static_cast<uint32_t>(ring_row[warp][get][rr + i * RP])) = *reinterpret_cast<const uint4*>(slot + copy_at(i));
      __syncwarp();
      get = (get + 1) % kRing;
      fetch();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
  }
}

template <typename Kernel>
static cudaError_t adapter_smem(Kernel kernel, int smem, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || smem <= 48 * 1024 || (dev < 64 && ready[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev < 64) ready[dev] = true;
  return e;
}

// Most entries of a list of `per` rows each: every adapter with a row has one, and what its other rows fill.
static int adapter_entries(int rows, int slots, int per) {
  const int used = min(slots + 1, rows);
  return used + (rows - used) / per;
}
static int adapter_items(int rows, int slots) { return adapter_entries(rows, slots, adapter_item_rows(rows)); }
static int adapter_strips(int rows, int slots) { return adapter_entries(rows, slots, 16); }

// CTAs that share k: as long as two find room on every SM.  A layer by the most CTAs: 256 rows, 240 over 60 adapters of rank 64 (one launch), 160 185 us, 320 133,
// 640 154; 48 rows, 36 over nine, 80 63 us, 160 and more 46; 8192 rows of rank 16 (tiles) 148 456 us, 320 408, 592 426.  Clusters of sixteen change nothing.
static int adapter_splits(int units, int k) {
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= 320 && k / (splits * 2) >= 256) splits *= 2;
  return splits;
}

template <int R16, int MT>
static cudaError_t adapter_few(const CbAdapter& p, int items, cudaStream_t stream) {
  const int rt = p.sections * R16 * 16, smem = (8 * 16 * 68 + 16 * rt) * 4 + 2 * 16 * (rt + 8) * 2;
  static_assert((8 * 16 * 68 + 16 * 512) * 4 + 2 * 16 * 520 * 2 <= 113 * 1024, "two of the largest on an SM");
  static int ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (smem > 48 * 1024 && (dev >= 64 || ready[dev] < smem)) {
    e = cudaFuncSetAttribute(adapter_few_kernel<R16, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev] = smem;
  }
  const int splits = adapter_splits(items, p.k);
  return launch(adapter_few_kernel<R16, MT>, dim3(min(items, 592 / splits) * splits), dim3(kAdapterThreads), smem, stream, dim3(splits, 1, 1), p, splits);
}

template <int NT>
static cudaError_t adapter_down_tile(const CbAdapter& p, int items, cudaStream_t stream) {
  constexpr int NR = NT * 16, smem = DownTile<NT>::kBytes;
  static_assert(64 * DownTile<NT>::SP * 4 <= smem, "the sums fit where the stages were");
  static bool ready[64] = {};
  const cudaError_t e = adapter_smem(adapter_down_tile_kernel<NT>, smem, ready);
  if (e != cudaSuccess) return e;
  const int units = items * ((p.sections * p.rank + NR - 1) / NR);
  const int splits = adapter_splits(units, p.k);
  return launch(adapter_down_tile_kernel<NT>, dim3(min(units, 592 / splits) * splits), dim3(kAdapterThreads), smem, stream, dim3(splits, 1, 1), p, splits);
}

template <int R16, int MT>
static cudaError_t adapter_up(const CbAdapter& p, cudaStream_t stream) {
  constexpr int smem = 8 * 4 * 512 * MT, resident = R16 * MT <= 4 ? 3 : 2;
  static bool ready[64] = {};
  const cudaError_t e = adapter_smem(adapter_up_kernel<R16, MT>, smem, ready);
  if (e != cudaSuccess) return e;
  const int warps = adapter_strips(p.rows, p.slots) * ((p.n + 16 * MT - 1) / (16 * MT));
  return launch(adapter_up_kernel<R16, MT>, dim3(min((warps + 7) / 8, 148 * resident)), dim3(kAdapterThreads), smem, stream, p);
}

template <int R16>
static int adapter_launch(const CbAdapter& p, cudaStream_t stream) {
  bool wide = R16 < 4;                                                // a warp's columns belong to one section
  for (int i = 0; i + 1 < p.sections; ++i) wide = wide && p.width[i] % 64 == 0;
  constexpr int kWide = R16 < 4 ? 4 : 2;
  const int items = adapter_items(p.rows, p.slots);
  if (p.rows <= kAdapterFewRows) return static_cast<int>(wide ? adapter_few<R16, kWide>(p, items, stream) : adapter_few<R16, 2>(p, items, stream));
  const int n = p.sections * R16;                                     // sixteens of ranks
  const cudaError_t e = n == 1 ? adapter_down_tile<1>(p, items, stream) : n == 2 ? adapter_down_tile<2>(p, items, stream) : n == 3 ? adapter_down_tile<3>(p, items, stream)
                      : n == 4 ? adapter_down_tile<4>(p, items, stream) : n % 8 == 0 ? adapter_down_tile<8>(p, items, stream) : adapter_down_tile<6>(p, items, stream);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(wide ? adapter_up<R16, kWide>(p, stream) : adapter_up<R16, 2>(p, stream));
}

}  // namespace cb

extern "C" {

int cb_adapter_rows(const void* ids, int rows, int slots, void* order, void* items, void* strips, void* stream) {
  using namespace cb;
  if (rows < 0 || rows > kAdapterMaxRows || slots < 1 || slots > kAdapterMaxSlots) return -10;
  constexpr int most = 32 * (kAdapterMaxSlots + 1) * sizeof(unsigned short);
  const int smem = 32 * (slots + 1) * static_cast<int>(sizeof(unsigned short));
  static bool ready[64] = {};                                         // once a device, whatever the size: the kernel's own arrays (12.5 KB) count towards the usual 48 KB too
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) e = cudaFuncSetAttribute(adapter_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 64) ready[dev] = true;
  return static_cast<int>(launch(adapter_rows_kernel, dim3(1), dim3(kSortThreads), smem, static_cast<cudaStream_t>(stream), static_cast<const int*>(ids), rows, slots,
                                 static_cast<int*>(order), static_cast<int*>(items), static_cast<int*>(strips)));
}

int cb_adapter_add(const CbAdapter* p, void* stream) {
  using namespace cb;
  if (p->rows < 0 || p->rows > kAdapterMaxRows || p->slots < 1 || p->slots > kAdapterMaxSlots || p->k < 8 || p->k % 8 || p->n < 8 || p->n % 8) return -10;
  if (p->sections < 1 || p->sections > kAdapterSections || p->ldx % 8 || p->ldy % 8 || p->ldo % 8 || p->ldy > kAdapterMaxStride || p->ldo > kAdapterMaxStride) return -11;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->rank) {
    case 16: return adapter_launch<1>(*p, s);
    case 32: return adapter_launch<2>(*p, s);
    case 64: return adapter_launch<4>(*p, s);
    case 128: return adapter_launch<8>(*p, s);
  }
  return -14;
}

}  // extern "C"
