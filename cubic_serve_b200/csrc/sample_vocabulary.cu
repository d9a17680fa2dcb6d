// A draw from the whole vocabulary: temperature, top-k, top-p and min-p of each row, from a uniform number.
//
// A row's tokens in order (value descending, id ascending) have weights w = exp((x - max) / T).  The row keeps a prefix of that order: the first k;
// of those the shortest prefix with at least p of their mass; of those the tokens with w >= m.  The draw is the first token whose running
// mass is above u times the mass kept.  Only prefixes matter, so nothing is sorted: a prefix is found in a histogram.
//
// A row's values fall into bins of one sign, exponent and seven bits of mantissa: for bf16 a bin IS a value.  48 exponents have bins (2^-32 to 2^16, or those
// below the row's largest magnitude that matters); smaller magnitudes share the bin of zero.  bf16: counts alone are gathered, a weight is computed once a
// bin, in 64 bits.  fp32: counts and masses, and the bin that holds the end of a prefix is divided again by the bits below, as is the bin of zero if it holds
// anything else.
// Masses are whole multiples of 2^-42 of the largest weight: sums of 64-bit integers do not depend on their order, and two equal rows draw the same.
//
// Bound by the histogram's additions in shared memory, then by what is read: 2 bytes a token and, for the id, a second look at the row, which is in L2.
#include "ptx.cuh"
#include "launch.cuh"
#include "philox.cuh"

// Mirrored by ops/native.py::VocabularyStruct.
struct CbVocabulary {
  const void* logits; long long ld;          // [rows, vocab], bf16 or fp32
  const uint32_t* mask; long long ld_mask;   // [rows, words] allowed tokens, or null
  const float* temperature;                  // [rows], 0: greedy
  const int* top_k; const float* top_p; const float* min_p;      // [rows] or null; 0, 1, 0: none
  const float* uniforms;                     // [rows], or null: seeds and counters
  const unsigned long long* seeds; const unsigned long long* counters;
  const int* rows_of;                        // [rows] row r is row rows_of[r] of everything (below 0: none), or null: r
  int* ids; float* logprob; int* kept;       // [rows]; the last two or null
  int rows, vocab, f32;
};

namespace cb {

typedef unsigned long long u64;

static constexpr int kVocabThreads = 512;
static constexpr int kVocabMax = 1 << 20;
static constexpr int kSpan = 48 * 128;                     // bins of a sign
static constexpr int kZero = kSpan + 1;                    // bin of zero; the last one at either end is for what is larger
static constexpr int kBins = 2 * kSpan + 3;
static constexpr int kRun = (kBins + kVocabThreads - 1) / kVocabThreads;
static constexpr double kUnit = 4398046511104.0;           // 2^42
static constexpr float kLeastMinP = 8.6736174e-19f;        // 2^-60: less is as good as none

__device__ __forceinline__ uint32_t sort_key(uint32_t u) {                 // order of the values; both zeros are one
  if ((u << 1) == 0) return 0x80000000u;
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ int bin_of(uint32_t u, int base) {
  const int m = min(max(static_cast<int>((u & 0x7fffffffu) >> 16) - base, 0), kSpan + 1);
  return static_cast<int>(u) < 0 ? kZero - m : kZero + m;
}
// The keys of a bin.
__device__ __forceinline__ void bin_keys(int bin, int base, uint32_t& lo, uint32_t& hi) {
  const int m = abs(bin - kZero);
  const uint32_t least = m == 0 ? 0u : static_cast<uint32_t>(base + m) << 16;
  const uint32_t most = m == 0 ? (static_cast<uint32_t>(base) << 16 | 0xffffu) : m <= kSpan ? (least | 0xffffu) : 0x7f800000u;
  if (m == 0) { lo = ~(0x80000000u | most); hi = 0x80000000u | most; }
  else if (bin > kZero) { lo = 0x80000000u | least; hi = 0x80000000u | most; }
  else { lo = ~(0x80000000u | most); hi = ~(0x80000000u | least); }
}

// A row's tokens, eight neighbours at a time from a 16-byte boundary.
template <bool F32>
struct VocabRow {
  const char* base;
  const uint32_t* mask;
  int shift, vocab, vectors, words;

  __device__ __forceinline__ VocabRow(const CbVocabulary& p, size_t row) {
    constexpr int E = F32 ? 4 : 2;
    const char* at = static_cast<const char*>(p.logits) + row * p.ld * E;
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
    base = at - skew;
    shift = skew / E;
    vocab = p.vocab;
    vectors = (vocab + shift + 7) >> 3;
    mask = p.mask ? p.mask + row * p.ld_mask : nullptr;
    words = (vocab + 31) >> 5;
  }
  __device__ __forceinline__ int first(int v) const { return v * 8 - shift; }
  __device__ __forceinline__ uint32_t word(int w) const { return w >= 0 && w < words ? __ldg(mask + w) : 0u; }
  // the bits of the values, and which of them count: tokens of the row that the mask allows and that are more than -inf
  __device__ __forceinline__ uint32_t load(int v, uint32_t (&u)[8]) const {
    const int i = first(v);
    uint32_t ok = 0xffu;
    if (i >= 0 && i + 8 <= vocab) {
      if (F32) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(base) + v * 2), b = __ldg(reinterpret_cast<const uint4*>(base) + v * 2 + 1);
        u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w; u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
      } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(base) + v);
        u[0] = a.x << 16; u[1] = a.x & 0xffff0000u; u[2] = a.y << 16; u[3] = a.y & 0xffff0000u;
        u[4] = a.z << 16; u[5] = a.z & 0xffff0000u; u[6] = a.w << 16; u[7] = a.w & 0xffff0000u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = i + j >= 0 && i + j < vocab;
        if (!in) ok &= ~(1u << j);
        u[j] = !in ? 0u : F32 ? __ldg(reinterpret_cast<const uint32_t*>(base) + v * 8 + j) : static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(base) + v * 8 + j)) << 16;
      }
    }
    if (mask) {
      const int w = i >> 5;
      ok &= __funnelshift_r(word(w), (i & 31) > 24 ? word(w + 1) : 0u, i & 31);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((u[j] & 0x7fffffffu) > 0x7f800000u || u[j] == 0xff800000u) ok &= ~(1u << j);
    return ok;
  }
};

struct VocabScratch {
  u64 sum_m[kVocabThreads / 32];
  int sum_c[kVocabThreads / 32];
  int mixed;                                 // bf16: the bin of zero holds other values
  u64 zero_m;                                // and their mass
  // what a search found: the prefix before, the values it ended in, how many there are and their weight
  int before_c, ties;
  u64 before_m;
  uint32_t lo, hi;
  int bin;
  u64 sub_m[256];
  int sub_c[256];
};

// Beside an infinity nothing else has weight, at an infinite temperature either.
__device__ __forceinline__ double weight(uint32_t key, float best, double t) {
  const float v = key_value(key);
  return v == best ? 1.0 : best == INFINITY ? 0.0 : exp((static_cast<double>(v) - best) / t);
}

template <bool F32>
struct VocabSearch {
  const VocabRow<F32>& row;
  VocabScratch& s;
  const int* count; const u64* mass;            // by bin, descending
  int base;
  float best;
  double t;
  int run_c; u64 run_m; int pre_c; u64 pre_m;   // the thread's run of bins and what is before it

  __device__ __forceinline__ uint32_t value_of(int bin) const {                 // key of a bf16 bin's value
    uint32_t lo, hi;
    bin_keys(bin, base, lo, hi);
    return bin == kZero ? 0x80000000u : bin > kZero ? lo : hi;
  }
  __device__ __forceinline__ bool many(int bin) const { return F32 || (bin == kZero && s.mixed); }     // a bin of several values
  __device__ __forceinline__ u64 bin_mass(int bin) const {
    if (F32) return mass[bin];
    if (many(bin)) return s.zero_m;
    const int c = count[bin];
    return c == 0 || bin == 0 ? 0ull : static_cast<u64>(__double2ll_rn(c * (weight(value_of(bin), best, t) * kUnit)));
  }
  // The first prefix with at least `want` tokens, or `by_mass` with a mass of at least `want`.  In a scratch that all threads may read.
  __device__ void find(bool by_mass, u64 want) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (by_mass ? pre_m < want && want <= pre_m + run_m : static_cast<u64>(pre_c) < want && want <= static_cast<u64>(pre_c) + run_c) {
      int c = pre_c;
      u64 m = pre_m;
      for (int i = 0; i < kRun; ++i) {
        const int bin = kBins - 1 - (tid * kRun + i);
        if (bin < 0) break;
        const int bc = count[bin];
        if (bc == 0) continue;
        const u64 bm = bin_mass(bin);
        s.before_c = c; s.before_m = m; s.bin = bin; s.ties = bc;
        bin_keys(bin, base, s.lo, s.hi);
        if (by_mass ? m + bm >= want : static_cast<u64>(c) + bc >= want) break;
        c += bc;
        m += bm;
      }
    }
    __syncthreads();
    if (many(s.bin)) refine(by_mass, want);
  }
  // Divides what a search ended in until it is one value.
  __device__ void refine(bool by_mass, u64 want) {
    const int tid = threadIdx.x;
    while (s.lo != s.hi) {
      const uint32_t lo = s.lo, hi = s.hi;
      const int shift = max(0, 24 - __clz(hi - lo));
      for (int i = tid; i < 256; i += kVocabThreads) { s.sub_c[i] = 0; s.sub_m[i] = 0; }
      __syncthreads();
      for (int v = tid; v < row.vectors; v += kVocabThreads) {
        uint32_t u[8];
        const uint32_t ok = row.load(v, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = sort_key(u[j]);
          if (!(ok >> j & 1) || k < lo || k > hi) continue;
          atomicAdd(&s.sub_c[(k - lo) >> shift], 1);
          atomicAdd(&s.sub_m[(k - lo) >> shift], static_cast<u64>(__double2ll_rn(weight(k, best, t) * kUnit)));
        }
      }
      __syncthreads();
      if (tid == 0) {
        int c = s.before_c, i = 255;
        u64 m = s.before_m;
        for (; i > 0; --i) {
          if (by_mass ? m + s.sub_m[i] >= want : static_cast<u64>(c) + s.sub_c[i] >= want) break;
          c += s.sub_c[i];
          m += s.sub_m[i];
        }
        s.before_c = c; s.before_m = m; s.ties = s.sub_c[i];
        s.lo = lo + (static_cast<uint32_t>(i) << shift);
        s.hi = min(hi, s.lo + ((1u << shift) - 1));
      }
      __syncthreads();
    }
  }
  // weight of the tokens that a search ended in, in units
  __device__ __forceinline__ double found_weight() const {
    if (many(s.bin)) return static_cast<double>(__double2ll_rn(weight(s.lo, best, t) * kUnit));
    return s.bin == 0 ? 0.0 : weight(value_of(s.bin), best, t) * kUnit;
  }
};

// The thread's run of bins, and what is before it.
template <bool F32>
__device__ void vocab_runs(VocabSearch<F32>& f, int& total_c, u64& total_m) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int c = 0;
  u64 m = 0;
  for (int i = 0; i < kRun; ++i) {
    const int bin = kBins - 1 - (tid * kRun + i);
    if (bin < 0) break;
    c += f.count[bin];
    m += f.bin_mass(bin);
  }
  f.run_c = c;
  f.run_m = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, c, o);
    const u64 b = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) { c += a; m += b; }
  }
  __syncthreads();
  if (lane == 31) { f.s.sum_c[warp] = c; f.s.sum_m[warp] = m; }
  __syncthreads();
  total_c = 0;
  total_m = 0;
  for (int w = 0; w < kVocabThreads / 32; ++w) {
    if (w == warp) { f.pre_c = total_c + c - f.run_c; f.pre_m = total_m + m - f.run_m; }
    total_c += f.s.sum_c[w];
    total_m += f.s.sum_m[w];
  }
}

template <bool F32>
__global__ void __launch_bounds__(kVocabThreads, F32 ? 1 : 2)
sample_vocabulary_kernel(const CbVocabulary p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ VocabScratch s;
  __shared__ uint32_t top_key[kVocabThreads / 32];
  u64* mass = reinterpret_cast<u64*>(dyn);
  int* count = reinterpret_cast<int*>(dyn + (F32 ? kBins * sizeof(u64) : 0));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int r = p.rows_of ? p.rows_of[blockIdx.x] : blockIdx.x;
  if (r < 0) return;
  const VocabRow<F32> row(p, r);
  const float temp = p.temperature ? p.temperature[r] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double t = greedy ? 1.0 : static_cast<double>(temp);
  int base = ((127 - 32) << 7) - 1;

  // bf16: counts and the largest value in one look.  fp32: the largest first, for the masses.
  uint32_t best_key = 0;
  for (int look = 0; look < 2; ++look) {
    const bool fill = !greedy && (!F32 || look == 1);
    if (fill) {
      for (int i = tid; i < kBins; i += kVocabThreads) { count[i] = 0; if (F32) mass[i] = 0; }
      if (tid == 0) { s.mixed = 0; s.zero_m = 0; }
      __syncthreads();
    }
    if (F32 && look == 1) {
      const float best = key_value(best_key);
      for (int v = tid; v < row.vectors; v += kVocabThreads) {
        uint32_t u[8];
        const uint32_t ok = row.load(v, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!(ok >> j & 1)) continue;
          const int b = bin_of(u[j], base);
          atomicAdd(&count[b], 1);
          atomicAdd(&mass[b], static_cast<u64>(__double2ll_rn(weight(sort_key(u[j]), best, t) * kUnit)));
        }
      }
      __syncthreads();
      break;
    }
    uint32_t top = 0;
#pragma unroll 2
    for (int v = tid; v < row.vectors; v += kVocabThreads) {
      uint32_t u[8];
      const uint32_t ok = row.load(v, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(ok >> j & 1)) continue;
        top = max(top, sort_key(u[j]));
        if (!F32 && fill) {
          const int b = bin_of(u[j], base);
          atomicAdd(&count[b], 1);
          if (b == kZero && (u[j] << 1)) s.mixed = 1;
        }
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) top_key[warp] = top;
    __syncthreads();
    best_key = 0;
    for (int w = 0; w < kVocabThreads / 32; ++w) best_key = max(best_key, top_key[w]);
    __syncthreads();
    if (greedy || best_key == 0) break;
    // The exponents that matter: up to the largest magnitude that a token of weight e^-44 or more can have.  Other than the usual ones: a second look.
    const double best = key_value(best_key), far = best - 44.0 * t, most = isinf(best) ? 1e300 : fmax(fabs(best), fabs(far));
    if (most < 1.0 || most >= 65536.0) {
      const int e = most >= 3e38 ? (isinf(best) ? 128 : 127) : most < 1e-37 ? -126 : ilogb(most);
      base = max(0, ((e - 47 + 127) << 7) - 1);
    } else if (!F32) {
      break;
    }
  }

  if (best_key == 0) {                          // nothing may be drawn
    if (tid == 0) {
      p.ids[r] = 0;
      if (p.logprob) p.logprob[r] = -INFINITY;
      if (p.kept) p.kept[r] = 0;
    }
    return;
  }
  uint32_t pick_key = best_key;
  int pick = 0;                                 // which of the tokens of that value, by id
  if (!greedy) {
    VocabSearch<F32> f{row, s, count, mass, base, key_value(best_key), t, 0, 0ull, 0, 0ull};
    if (!F32 && s.mixed) {
      u64 m = 0;
      for (int v = tid; v < row.vectors; v += kVocabThreads) {
        uint32_t u[8];
        const uint32_t ok = row.load(v, u);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((ok >> j & 1) && bin_of(u[j], base) == kZero) m += static_cast<u64>(__double2ll_rn(weight(sort_key(u[j]), f.best, t) * kUnit));
      }
      if (m) atomicAdd(&s.zero_m, m);
      __syncthreads();
    }
    int total;
    u64 sum;
    vocab_runs(f, total, sum);
    int n = total;
    u64 kept = sum;
    const int k = p.top_k ? p.top_k[r] : 0;
    const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
    auto mass_of = [&](int prefix) {            // of the prefix that the last search ended in
      return s.before_m + static_cast<u64>(__double2ll_rn((prefix - s.before_c) * f.found_weight()));
    };
    if (k > 0 && k < n) {
      f.find(false, k);
      n = k;
      kept = mass_of(n);
    }
    if (tp < 1.f) {
      const u64 want = max(1ull, static_cast<u64>(ceil(static_cast<double>(fmaxf(tp, 0.f)) * static_cast<double>(kept))));
      f.find(true, want);
      const double w = f.found_weight();
      const int m = min(s.ties, max(1, static_cast<int>(ceil(static_cast<double>(want - s.before_m) / w))));
      if (s.before_c + m < n) {
        n = s.before_c + m;
        kept = mass_of(n);
      }
    }
    if (mp >= kLeastMinP) {
      const double least = fmin(static_cast<double>(mp), 1.0);
      int c = 0;
      if (F32 || s.mixed) {
        for (int v = tid; v < row.vectors; v += kVocabThreads) {
          uint32_t u[8];
          const uint32_t ok = row.load(v, u);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (ok >> j & 1) c += weight(sort_key(u[j]), f.best, t) >= least;
        }
      } else {
        for (int i = 0; i < kRun; ++i) {
          const int bin = kBins - 1 - (tid * kRun + i);
          if (bin <= 0) break;
          if (count[bin] && weight(f.value_of(bin), f.best, t) >= least) c += count[bin];
        }
      }
      c = __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
      if (lane == 0) s.sum_c[warp] = c;
      __syncthreads();
      c = 0;
      for (int w = 0; w < kVocabThreads / 32; ++w) c += s.sum_c[w];
      c = max(c, 1);
      if (c < n) {
        n = c;
        f.find(false, n);
        kept = mass_of(n);
      }
    }
    float u = p.uniforms ? p.uniforms[r] : philox_uniform(p.seeds ? p.seeds[r] : 0ull, p.counters ? p.counters[r] : 0ull);
    u = fminf(fmaxf(u, 0.f), 0.99999994f);
    const double aim = static_cast<double>(u) * static_cast<double>(kept);
    f.find(true, static_cast<u64>(aim) + 1);
    const double w = f.found_weight();
    pick = w > 0.0 ? static_cast<int>((aim - static_cast<double>(s.before_m)) / w) : 0;
    pick = max(0, min(pick, min(s.ties, n - s.before_c) - 1));
    pick_key = f.many(s.bin) ? s.lo : f.value_of(s.bin);
    if (tid == 0) {
      const float v = key_value(pick_key);
      if (p.logprob) p.logprob[r] = static_cast<float>((v == f.best ? 0.0 : (static_cast<double>(v) - f.best) / t) - log(static_cast<double>(kept) / kUnit));
      if (p.kept) p.kept[r] = n;
    }
  } else if (tid == 0) {
    if (p.logprob) p.logprob[r] = 0.f;
    if (p.kept) p.kept[r] = 1;
  }

  // the token: how many of the value are in every tile, then a look at the tile that holds it
  __syncthreads();
  const int tiles = (row.vectors + 31) >> 5;
  unsigned short* in_tile = reinterpret_cast<unsigned short*>(dyn);
  for (int i = warp; i < tiles; i += kVocabThreads / 32) {
    const int v = i * 32 + lane;
    int c = 0;
    if (v < row.vectors) {
      uint32_t u[8];
      const uint32_t ok = row.load(v, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) c += (ok >> j & 1) && sort_key(u[j]) == pick_key;
    }
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) in_tile[i] = static_cast<unsigned short>(c);
  }
  __syncthreads();
  if (warp != 0) return;
  int tile = -1;
  for (int i0 = 0; i0 < tiles; i0 += 32) {
    const int c = i0 + lane < tiles ? in_tile[i0 + lane] : 0;
    int upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += a;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, upto > pick);
    if (past) {
      const int l = __ffs(past) - 1;
      tile = i0 + l;
      pick -= __shfl_sync(0xffffffffu, upto - c, l);
      break;
    }
    pick -= __shfl_sync(0xffffffffu, upto, 31);
  }
  if (tile < 0) return;
  const int v = tile * 32 + lane;
  uint32_t hit = 0;
  if (v < row.vectors) {
    uint32_t u[8];
    const uint32_t ok = row.load(v, u);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((ok >> j & 1) && sort_key(u[j]) == pick_key) hit |= 1u << j;
  }
  int upto = __popc(hit);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += a;
  }
  int mine = pick - (upto - __popc(hit));
  if (mine >= 0 && mine < __popc(hit)) {
    while (mine-- > 0) hit &= hit - 1;
    p.ids[r] = row.first(v) + __ffs(hit) - 1;
  }
}

}  // namespace cb

extern "C" int cb_sample_vocabulary(const CbVocabulary* p, void* stream) {
  using namespace cb;
  if (p->rows < 0 || p->vocab < 1 || p->vocab > kVocabMax || p->ld < p->vocab || (p->mask && p->ld_mask * 32 < p->vocab)) return -10;
  if (reinterpret_cast<uintptr_t>(p->logits) % (p->f32 ? 4 : 2)) return -11;
  if (p->rows == 0) return 0;
  const int smem = kBins * (p->f32 ? sizeof(u64) + sizeof(int) : sizeof(int));
  const void* kernel = p->f32 ? reinterpret_cast<const void*>(sample_vocabulary_kernel<true>) : reinterpret_cast<const void*>(sample_vocabulary_kernel<false>);
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return static_cast<int>(p->f32 ? launch(sample_vocabulary_kernel<true>, dim3(p->rows), dim3(kVocabThreads), smem, st, *p)
                                 : launch(sample_vocabulary_kernel<false>, dim3(p->rows), dim3(kVocabThreads), smem, st, *p));
}
