// A draw from the whole vocabulary: temperature, top-k, top-p and min-p of each row, from a uniform number.
//
// A row's tokens in order (value descending, id ascending) have weights w = exp((x - max) / T).  The row keeps a prefix of that order: the first k;
// of those the shortest prefix with at least p of their mass; of those the tokens with w >= m.  The draw is the first token whose running
// mass is above u times the mass kept.  Only prefixes matter, so nothing is sorted: a prefix is found in a histogram.
//
// A row's values fall into bins of one sign, exponent and seven bits of mantissa: for bf16 a bin IS a value.  48 exponents have bins (2^-32 to 2^16, or those
// below the row's largest magnitude that matters); smaller magnitudes share the bin of zero.  bf16: counts alone are gathered, a weight is computed once a
// bin, in 64 bits.  fp32: counts and masses, and the bin that holds the end of a prefix is divided again by the bits below, as is the bin of zero if it holds
// anything else.  Masses are whole multiples of 2^-42 of the largest weight: sums of 64-bit integers do not depend on their order, so
// that a launch repeats itself bit for bit.
//
// A row belongs to one CTA or to a cluster of up to eight, each with a share of its tokens: tables are added up through the peers' shared memory.
//
// Few rows are bound by latency, many by additions to shared memory: one a token, about 5 cycles a warp of 32.  One row of 151936 bf16 values takes 16 us: the look
// 4, its tables and their sums 5, the search and the id 3, the launch 3.  48 rows with masks and all filters 28: the look 10.  256 rows with top-p 50, 1.6 TB/s: an
// SM with one row is through its look after 12 us, one with two after 27; sums 5, each search 1 to 2, the id 1.  Nine fp32 rows of 50257 with all filters 39: a look
// for the largest 2, one with masses 4, sums 7, each of four searches 5.  (Exponentials are no burden: without them the look takes 2.5.)
#include "ptx.cuh"
#include "launch.cuh"
#include "philox.cuh"

// Packed by ops/native.py::VOCABULARY.
struct CbVocabulary {
  const void* logits; long long ld;          // [rows, vocab], bf16 or fp32
  const uint32_t* mask; long long ld_mask;   // [rows, words] allowed tokens, or null; a stride of 0: of all rows
  const float* temperature;                  // [rows], 0: greedy
  const int* top_k; const float* top_p; const float* min_p;      // [rows] or null; 0, 1, 0: none
  const float* uniforms;                     // [rows], or null: seeds and counters
  const unsigned long long* seeds; const unsigned long long* counters;
  const int* rows_of;                        // [rows] row r is row rows_of[r] of everything (below 0: none), or null: r
  int* ids; float* logprob; int* kept;       // [rows]; the last two or null
  int rows, vocab, f32;
  int limit;                                 // rows of every tensor: one of rows_of that is not below it is none
};

namespace cb {

typedef unsigned long long u64;

// A table with masses leaves room for one CTA on an SM, so it has all the threads: 48 rows of 151936 tokens with all filters take 136 us, with 512 threads 162.
template <bool F32> constexpr int kThreadsOf = F32 ? 1024 : 512;
static constexpr int kVocabMostWarps = 32;
static constexpr int kVocabMax = 1 << 20;
static constexpr int kTeamMax = 8;                         // CTAs of a row
static constexpr int kSpan = 48 * 128;                     // bins of a sign; one more at the end for what is larger
static constexpr int kNegative = 8192;                     // where the bins of negative values start
static constexpr int kTable = kNegative + kSpan + 2;
// in descending order: kSpan + 1 positive bins, zero, as many negative ones
static constexpr int kZero = kSpan + 1, kBins = 2 * kSpan + 3;
// Segments of 32 bins, a lane each: what is too large, 4 an exponent down to zero, zero, and the same below it.
static constexpr int kSideSegments = kSpan / 32, kZeroSegment = kSideSegments + 1, kSegments = 2 * kSideSegments + 3;
static constexpr double kUnit = 4398046511104.0;           // 2^42
static constexpr float kLeastMinP = 8.6736174e-19f;        // 2^-60: less is as good as none
static constexpr int kUsualBase = ((127 - 32) << 7) - 1;
static_assert(kSegments <= kThreadsOf<false>, "a thread holds the sums before a segment");

// Places 1 to 32, 33 to 64, ... of either side are a segment: they start on 16 bytes.
static constexpr int kCountAt = 3, kMassAt = 1, kCountRoom = (kCountAt + kTable + 3) / 4 * 4, kMassRoom = (kMassAt + kTable + 1) / 2 * 2;
static constexpr int kFew = 256;                           // tokens of a bin that are ranked one against the other: a search takes 5 us, with two divisions 11

__device__ __forceinline__ uint32_t sort_key(uint32_t u) {                 // order of the values; both zeros are one
  if ((u << 1) == 0) return 0x80000000u;
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Place of a value in the table, of a descending bin in the table, and the keys of a bin.
__device__ __forceinline__ int place_of(uint32_t u, int base) {
  return min(max(static_cast<int>((u & 0x7fffffffu) >> 16) - base, 0), kSpan + 1) + (static_cast<int>(u) < 0 ? kNegative : 0);
}
__device__ __forceinline__ int place_of_bin(int d) { return d <= kZero ? kZero - d : kNegative + (d - kZero); }
__device__ __forceinline__ void bin_keys(int d, int base, uint32_t& lo, uint32_t& hi) {
  const int m = abs(d - kZero);
  const uint32_t least = m == 0 ? 0u : static_cast<uint32_t>(base + m) << 16;
  const uint32_t most = m == 0 ? (static_cast<uint32_t>(base) << 16 | 0xffffu) : m <= kSpan ? (least | 0xffffu) : 0x7f800000u;
  if (m == 0) { lo = ~(0x80000000u | most); hi = 0x80000000u | most; }
  else if (d < kZero) { lo = 0x80000000u | least; hi = 0x80000000u | most; }
  else { lo = ~(0x80000000u | most); hi = ~(0x80000000u | least); }
}

__device__ __forceinline__ int bin_in(int g, int lane) {                   // bin of a segment's lane, kBins: none
  if (g == 0 || g == kZeroSegment || g == kSegments - 1) return lane ? kBins : g == 0 ? 0 : g == kZeroSegment ? kZero : kBins - 1;
  return (g < kZeroSegment ? (g - 1) * 32 + 1 : (g - kZeroSegment - 1) * 32 + kZero + 1) + lane;
}
__device__ __forceinline__ uint32_t ld_peer(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld_peer64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_peer128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_peer64(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }

// Adds to 64 bits of shared memory by its halves, which have additions of their own (a sum of 64 bits is a loop of compare and swap).
__device__ __forceinline__ void add_shared(u64* at, u64 v) {
  unsigned* half = reinterpret_cast<unsigned*>(at);
  const unsigned lo = static_cast<unsigned>(v), before = atomicAdd(half, lo), hi = static_cast<unsigned>(v >> 32) + (before + lo < lo);
  if (hi) atomicAdd(half + 1, hi);
}

// Can be drawn: more than -inf.
__device__ __forceinline__ bool is_more(uint32_t u) { return __uint_as_float(u) > -INFINITY; }

// A CTA's share of a row's tokens, eight neighbours at a time from a 16-byte boundary.
template <bool F32>
struct VocabRow {
  const char* base;
  const uint32_t* mask;
  int shift, vocab, words, from, to;            // vectors [from, to)

  __device__ __forceinline__ VocabRow(const CbVocabulary& p, size_t row, int rank, int team) {
    constexpr int E = F32 ? 4 : 2;
    const char* at = static_cast<const char*>(p.logits) + row * p.ld * E;
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
    base = at - skew;
    shift = skew / E;
    vocab = p.vocab;
    mask = p.mask ? p.mask + row * p.ld_mask : nullptr;
    words = (vocab + 31) >> 5;
    const int vectors = (vocab + shift + 7) >> 3, share = ((vectors + team - 1) / team + 31) & ~31;
    from = min(vectors, rank * share);
    to = min(vectors, from + share);
  }
  __device__ __forceinline__ int first(int v) const { return v * 8 - shift; }
  __device__ __forceinline__ bool whole(int v) const { return first(v) >= 0 && first(v) + 8 <= vocab; }
  __device__ __forceinline__ uint32_t word(int w) const { return w >= 0 && w < words ? mask[w] : 0u; }
  __device__ __forceinline__ uint32_t allowed(int v) const {                 // by the mask
    if (!mask) return 0xffu;
    if (shift == 0) return reinterpret_cast<const unsigned char*>(mask)[v];     // eight neighbours are a byte
    const int i = first(v), w = i >> 5;
    return __funnelshift_r(word(w), (i & 31) > 24 ? word(w + 1) : 0u, i & 31) & 0xffu;
  }
  // a vector in two steps, so that several are on their way, and do not wait for their mask: its bytes, if it lies in the row, then
  // the bits of the values, and which of them are tokens of the row that the mask allows
  __device__ __forceinline__ void fetch(int v, bool in, uint4& a, uint4& b) const {
    if (!in || !whole(v)) return;
    a = reinterpret_cast<const uint4*>(base)[F32 ? v * 2 : v];
    if (F32) b = reinterpret_cast<const uint4*>(base)[v * 2 + 1];
  }
  __device__ __forceinline__ uint32_t values(int v, uint32_t ok, const uint4& a, const uint4& b, uint32_t (&u)[8]) const {
    const int i = first(v);
    if (whole(v)) {
      if (F32) {
        u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w; u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
      } else {
        u[0] = a.x << 16; u[1] = a.x & 0xffff0000u; u[2] = a.y << 16; u[3] = a.y & 0xffff0000u;
        u[4] = a.z << 16; u[5] = a.z & 0xffff0000u; u[6] = a.w << 16; u[7] = a.w & 0xffff0000u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = i + j >= 0 && i + j < vocab;
        if (!in) ok &= ~(1u << j);
        u[j] = !in ? 0u : F32 ? reinterpret_cast<const uint32_t*>(base)[v * 8 + j] : static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(base)[v * 8 + j]) << 16;
      }
    }
    return ok;
  }
  // fn(values, which of them are allowed) of the CTA's vectors, U of a thread on their way at a time
  template <int U, typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    constexpr int T = kThreadsOf<F32>;
    for (int v0 = from + threadIdx.x; v0 < to; v0 += U * T) {
      uint4 a[U], b[U];
      uint32_t ok[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool in = v0 + k * T < to;
        fetch(v0 + k * T, in, a[k], b[k]);
        ok[k] = in ? allowed(v0 + k * T) : 0u;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (ok[k] == 0) continue;
        uint32_t u[8];
        const uint32_t in = values(v0 + k * T, ok[k], a[k], b[k], u);
        fn(u, in);
      }
    }
  }
};

// What the CTAs of a row tell one another; entry r is CTA r's.
struct VocabTold {
  u64 top[kTeamMax];             // largest key, or largest positive bf16 << 32 and what its bins at zero and below all others hold
  u64 zero_m[kTeamMax];          // mass of the bin of zero, and whether it holds another value
  u64 ids[kTeamMax];             // tokens of the value drawn
  u64 least[kTeamMax];           // tokens of at least min-p
};

struct VocabScratch {
  VocabTold told;
  u64 seg_m[kSegments]; int seg_c[kSegments];       // of the row: sums of a segment, then those before it
  double seg_w[kSegments], ratio[49];               // weight of a segment's first bin; of neighbouring bins of an exponent, one to the other
  u64 sum_m[kVocabMostWarps]; int sum_c[kVocabMostWarps];
  uint32_t warp_top[kVocabMostWarps];
  int owner;
  u64 sub_m[2][256]; __align__(16) int sub_c[2][256];            // a bin divided, or its tokens; two, for the peers may still read one
  int few[2];
  u64 part_m[256]; int part_c[256];                 // the same of all CTAs
  u64 found_m; int found_c, found_ties, found_at;
};

template <bool F32, bool TEAM>
struct Vocab {
  static constexpr int kVocabThreads = kThreadsOf<F32>, kVocabWarps = kVocabThreads / 32, kAhead = F32 ? 2 : 4;      // vectors of a thread on their way
  VocabRow<F32> row;
  VocabScratch& s;
  int* count; u64* mass;                        // the table of the CTA's own tokens; in the segments that are its, once they are merged, of the row's
  short* tile_max;                              // bf16: largest of every 256 tokens as a signed 16-bit number: exact where it is not negative
  int rank, team, base;
  bool mixed;                                   // bf16: the bin of zero holds other values, or may
  u64 zero_mass;
  float best;
  double inv_t;
  // what the last search ended in: the prefix before, bin, keys, how many tokens
  int before_c, bin, ties, turn;
  u64 before_m;
  uint32_t lo, hi;

  __device__ __forceinline__ void meet() const {
    if (TEAM) cluster_sync_all(); else __syncthreads();
  }
  __device__ __forceinline__ void tell(u64* entry, u64 v) const {                        // entry `rank` of every CTA's
    if (!TEAM) entry[0] = v;
    else for (int r = 0; r < team; ++r) st_peer64(cluster_map(smem_u32(entry + rank), r), v);
  }
  __device__ __forceinline__ u64 told(const u64* entry) const {
    u64 v = 0;
    for (int r = 0; r < team; ++r) v += entry[r];
    return v;
  }
  __device__ __forceinline__ double weight(uint32_t key) const {                         // beside an infinity nothing else has weight
    const float v = key_value(key);
    return v == best ? 1.0 : best == INFINITY ? 0.0 : exp((static_cast<double>(v) - best) * inv_t);
  }
  __device__ __forceinline__ u64 units(uint32_t key) const { return static_cast<u64>(__double2ll_rn(weight(key) * kUnit)); }
  __device__ __forceinline__ bool many(int d) const { return F32 || (d == kZero && mixed); }       // a bin of several values
  __device__ __forceinline__ uint32_t value_of(int d) const {                            // key of a bf16 bin's value
    uint32_t l, h;
    bin_keys(d, base, l, h);
    return d == kZero ? 0x80000000u : d < kZero ? l : h;
  }
  __device__ __forceinline__ int at(const int* t, int i) const {
    if (!TEAM) return t[i];
    uint32_t v[kTeamMax], c = 0;                 // all on their way before the first is needed
#pragma unroll
    for (int r = 0; r < kTeamMax; ++r) v[r] = r < team ? ld_peer(cluster_map(smem_u32(t + i), r)) : 0u;
#pragma unroll
    for (int r = 0; r < kTeamMax; ++r) c += v[r];
    return static_cast<int>(c);
  }
  __device__ __forceinline__ u64 at(const u64* t, int i) const {
    if (!TEAM) return t[i];
    u64 v[kTeamMax], m = 0;
#pragma unroll
    for (int r = 0; r < kTeamMax; ++r) v[r] = r < team ? ld_peer64(cluster_map(smem_u32(t + i), r)) : 0ull;
#pragma unroll
    for (int r = 0; r < kTeamMax; ++r) m += v[r];
    return m;
  }
  // What the table holds of a segment's bin, once merged: TEAM: at the CTA that the segment belongs to.
  __device__ __forceinline__ int merged(const int* t, int g, int i) const { return TEAM ? static_cast<int>(ld_peer(cluster_map(smem_u32(t + i), g % team))) : t[i]; }
  __device__ __forceinline__ u64 merged(const u64* t, int g, int i) const { return TEAM ? ld_peer64(cluster_map(smem_u32(t + i), g % team)) : t[i]; }
  __device__ __forceinline__ int bin_count(int g, int d) const {
    if (d >= kBins) return 0;
    return merged(count, g, place_of_bin(d)) + (d == kZero ? merged(count, g, kNegative) : 0);
  }
  // The values of a segment's bins fall by the same step of 2^(exponent - 7): their weights are the first one's times powers of one ratio.  387 + 49 exponentials
  // a row, a thread each, in place of one a bin.  In the segment of the best value the weights start from it.
  __device__ __forceinline__ uint32_t segment_mag(int g) const {             // magnitude, in bf16, of a segment's first bin
    return base + (g < kZeroSegment ? kSpan - (g - 1) * 32 : (g - kZeroSegment - 1) * 32 + 1);
  }
  __device__ __forceinline__ int segment_step(int g) const {                 // exponent of its steps, from that of the smallest bins
    const int mag = static_cast<int>(segment_mag(g)) - (g < kZeroSegment ? 1 : 0);
    return max(mag >> 7, 1) - max((base + 1) >> 7, 1);
  }
  __device__ __forceinline__ float segment_top(int g) const {                // its first value, the largest
    if (g == 0) return INFINITY;
    if (g == kZeroSegment) return 0.f;
    if (g == kSegments - 1) return -INFINITY;
    const uint32_t mag = segment_mag(g);
    return mag >= 0x7f80u ? (g < kZeroSegment ? INFINITY : -INFINITY) : __uint_as_float(mag << 16 | (g < kZeroSegment ? 0u : 0x80000000u));
  }
  __device__ __forceinline__ void weigh_segments() {
    const int tid = threadIdx.x;
    if (F32) return;
    if (tid < kSegments) {
      const float v = segment_top(tid);
      s.seg_w[tid] = v < best && best < INFINITY ? exp((static_cast<double>(v) - best) * inv_t) : -1.0;
    } else if (tid - kSegments < 49) {
      s.ratio[tid - kSegments] = exp(-ldexp(inv_t, max((base + 1) >> 7, 1) + (tid - kSegments) - 134));
    }
    __syncthreads();
  }
  // Of a segment that begins at the best value or above it: the best one's bin, 32 or more if that is in another segment.
  __device__ __forceinline__ int best_lane(int g) const {
    const int off = static_cast<int>(__float_as_uint(best) >> 16 & 0x7fffu) - static_cast<int>(segment_mag(g)), at = g < kZeroSegment ? -off : off;
    return (best < 0.f) != (g > kZeroSegment) || at < 0 ? 32 : at;
  }
  // mass of the bin of a segment's lane that holds c tokens
  __device__ __forceinline__ u64 lane_mass(int g, int lane, int c) const {
    const int d = bin_in(g, lane);
    if (F32) return d >= kBins ? 0ull : merged(mass, g, place_of_bin(d)) + (d == kZero ? merged(mass, g, kNegative) : 0ull);
    if (g == kSegments - 1) return 0;
    if (g == kZeroSegment && mixed) return c ? zero_mass : 0ull;
    double w = s.seg_w[g];
    if (g == kZeroSegment) {
      w = w < 0.0 ? (best == 0.f ? 1.0 : 0.0) : w;
    } else {
      int n = lane;
      if (w < 0.0) {
        n -= best_lane(g);
        w = n >= 0 ? 1.0 : 0.0;
      }
      double q = s.ratio[segment_step(g)];
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        if (n > 0 && (n >> i & 1)) w *= q;
        q *= q;
      }
    }
    return c ? static_cast<u64>(__double2ll_rn(c * (w * kUnit))) : 0ull;
  }

  // A thread's segment.
  __device__ __forceinline__ void segment_sum(int g) {
    const int lane = threadIdx.x & 31;
    const bool one = bin_in(g, 1) >= kBins;                      // a segment of one bin
    int from = 0, n = 0;
    double w0 = 0.0, q = 0.0, w = 0.0;
    u64 m = 0;
    if (!F32 && !one) {
      w0 = s.seg_w[g];
      q = s.ratio[segment_step(g)];
      if (w0 < 0.0) {                                            // up to the best value, whose weight is one; what is above it is empty
        from = best_lane(g);
        w0 = from < 32 ? 1.0 : 0.0;
      }
      if (lane >= from) {
        w = w0;
        double power = q;
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          if ((lane - from) >> i & 1) w *= power;
          power *= power;
        }
      }
    }
    const int d0 = bin_in(g, 0), place = place_of_bin(d0), step = d0 < kZero ? -1 : 1;
    if (one) {
      n = bin_count(g, d0);
      m = lane_mass(g, 0, n);
    } else {
#pragma unroll 8
      for (int i = 0; i < 32; ++i) {
        const int l = (i + lane) & 31, c = count[place + step * l];
        n += c;
        if (F32) {
          m += mass[place + step * l];
        } else {
          if (c) m += static_cast<u64>(__double2ll_rn(c * (w * kUnit)));
          w = ((l + 1) & 31) == from ? w0 : l == 31 ? 0.0 : w * q;
        }
      }
    }
    if (!TEAM) {
      s.seg_c[g] = n;
      s.seg_m[g] = m;
    } else {
      for (int r = 0; r < team; ++r) {
        st_cluster_u32(cluster_map(smem_u32(s.seg_c + g), r), n);
        st_peer64(cluster_map(smem_u32(s.seg_m + g), r), m);
      }
    }
  }

  // TEAM: the CTA adds the peers' tables to its own in every team-th segment, 16 bytes a load; the peers read nothing of these.  Masses come after the
  // counts, of bins that hold a token: most do not.
  template <typename V>
  __device__ __forceinline__ void merge(V* table) {
    constexpr int E = 16 / sizeof(V), L = 32 / E, P = 32 / L;                  // entries of a load, lanes of a segment, segments of a warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i0 = warp * P; i0 * team + rank < kSegments; i0 += kVocabWarps * P) {
      const int g = (i0 + lane / L) * team + rank;
      if (g >= kSegments) continue;
      const int d0 = bin_in(g, 0);
      if (bin_in(g, 1) < kBins) {
        const int at0 = (d0 < kZero ? place_of_bin(d0) - 31 : place_of_bin(d0)) + lane % L * E;
        if (sizeof(V) == 8 && (count[at0] | count[at0 + 1]) == 0) continue;
        V* own = table + at0;
        uint4 q[kTeamMax - 1];
#pragma unroll
        for (int r = 1; r < kTeamMax; ++r) {
          q[r - 1] = make_uint4(0, 0, 0, 0);
          if (r < team) q[r - 1] = ld_peer128(cluster_map(smem_u32(own), (rank + r) & (team - 1)));
        }
        V v[E];
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(own);
#pragma unroll
        for (int r = 1; r < kTeamMax; ++r) {
          const V* o = reinterpret_cast<const V*>(&q[r - 1]);
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] += o[e];
        }
        *reinterpret_cast<uint4*>(own) = *reinterpret_cast<const uint4*>(v);
      } else if (lane % L < (d0 == kZero ? 2 : 1)) {                           // a segment of one bin, two places for that of zero
        V* own = table + (lane % L ? kNegative : place_of_bin(d0));
        *own = at(own, 0);
      }
    }
  }
  // Sums of the segments, then those before each.  A thread takes a segment, from the bin of its lane on, so that 32 threads are at 32 banks; a CTA of several
  // takes every team-th segment.
  __device__ void sums(int& total_c, u64& total_m) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (TEAM) {
      merge(count);
      __syncthreads();
      if (F32) {
        merge(mass);
        __syncthreads();
      }
    }
    weigh_segments();
    if (tid * team + rank < kSegments) segment_sum(tid * team + rank);
    meet();
    const int own_c = tid < kSegments ? s.seg_c[tid] : 0;
    const u64 own_m = tid < kSegments ? s.seg_m[tid] : 0ull;
    int c = own_c;
    u64 m = own_m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, c, o);
      const u64 b = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) { c += a; m += b; }
    }
    if (lane == 31) { s.sum_c[warp] = c; s.sum_m[warp] = m; }
    __syncthreads();
    total_c = 0;
    total_m = 0;
#pragma unroll
    for (int w = 0; w < kVocabWarps; ++w) {
      if (w == warp) { pre_c = total_c + c - own_c; pre_m = total_m + m - own_m; }
      total_c += s.sum_c[w];
      total_m += s.sum_m[w];
    }
    end_c = pre_c + own_c;
    end_m = pre_m + own_m;
    if (tid < kSegments) { s.seg_c[tid] = pre_c; s.seg_m[tid] = pre_m; }
  }
  int pre_c, end_c; u64 pre_m, end_m;           // the thread's segment

  // The first prefix with at least `want` tokens, or `by_mass` with a mass of at least `want` (no more than there is).
  __device__ void find(bool by_mass, u64 want) {
    const int tid = threadIdx.x, lane = tid & 31;
    __syncthreads();
    if (by_mass ? pre_m < want && want <= end_m : static_cast<u64>(pre_c) < want && want <= static_cast<u64>(end_c)) s.owner = tid;
    __syncthreads();
    if (tid < 32) {
      const int g = s.owner, own_c = bin_count(g, bin_in(g, lane));
      settle(by_mass, want, own_c, lane_mass(g, lane, own_c), s.seg_c[g], s.seg_m[g]);
      if (lane == 0) s.found_at = bin_in(g, s.found_at);
    }
    __syncthreads();
    before_c = s.found_c; before_m = s.found_m; ties = s.found_ties; bin = s.found_at;
    bin_keys(bin, base, lo, hi);
    if (many(bin)) divide(by_mass, want);
  }
  // A warp's part of a search: the first lane at which the sums reach `want`.
  __device__ __forceinline__ void settle(bool by_mass, u64 want, int own_c, u64 own_m, int c0, u64 m0) {
    const int lane = threadIdx.x & 31;
    int c = own_c;
    u64 m = own_m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, c, o);
      const u64 b = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) { c += a; m += b; }
    }
    c += c0;
    m += m0;
    const uint32_t past = __ballot_sync(0xffffffffu, own_c && (by_mass ? m >= want : static_cast<u64>(c) >= want)), any = __ballot_sync(0xffffffffu, own_c);
    const int l = past ? __ffs(past) - 1 : 31 - __clz(any | 1u);
    if (lane == l) { s.found_c = c - own_c; s.found_m = m - own_m; s.found_ties = own_c; s.found_at = l; }
    __syncwarp();
  }
  // At least e^far of the best one's weight: without the exponential.
  __device__ __forceinline__ bool heavy_one(float v, double far) const { return v >= best || (best < INFINITY && (static_cast<double>(v) - best) * inv_t >= far); }
  // Tokens of a bf16 row that have at least `least` of the best one's weight: all in the segments before the last one whose first value has it, and
  // those of that one.
  __device__ int heavy(double least) {
    const int tid = threadIdx.x, lane = tid & 31;
    const double far = log(least);
    __syncthreads();
    if (tid < kSegments && heavy_one(segment_top(tid), far) && (tid + 1 == kSegments || !heavy_one(segment_top(tid + 1), far))) s.owner = tid;
    __syncthreads();
    if (tid < 32) {
      const int g = s.owner, d = bin_in(g, lane), c = bin_count(g, d);
      const int n = __reduce_add_sync(0xffffffffu, c && d < kBins - 1 && heavy_one(key_value(value_of(d)), far) ? c : 0);
      if (lane == 0) s.found_c = s.seg_c[g] + n;
    }
    __syncthreads();
    return s.found_c;
  }
  // Up to kFew tokens from lo to hi: every CTA gets them all, a thread each, and adds up those that come before its own.
  __device__ void settle_few(bool by_mass, u64 want) {
    const int tid = threadIdx.x;
    int* few = &s.few[turn];
    uint32_t* list = reinterpret_cast<uint32_t*>(s.sub_c[turn]);
    turn ^= 1;
    __syncthreads();
    if (tid == 0) *few = 0;
    __syncthreads();
    const float least = key_value(max(lo, 0x007fffffu)), most = key_value(min(hi, 0xff800000u));       // the bin of an infinity reaches behind it
    row.template each<kAhead>([&](const uint32_t (&u)[8], uint32_t ok) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = __uint_as_float(u[j]);
        if (!(v >= least && v <= most)) continue;
        const uint32_t k = sort_key(u[j]);                                     // the keys tell a range that ends below zero from one with it
        if (!(ok >> j & 1) || !is_more(u[j]) || k < lo || k > hi) continue;
        const int at = atomicAdd(few, 1);
        if (at < kFew) list[at] = k;
      }
    });
    meet();
    uint32_t key = 0;
    u64 own = 0;
    if (tid < ties) {
      int r = 0, i = tid;
      if (TEAM) {
        uint32_t n[kTeamMax];
#pragma unroll
        for (int q = 0; q < kTeamMax; ++q) n[q] = q < team ? ld_peer(cluster_map(smem_u32(few), q)) : 0u;
#pragma unroll
        for (int q = 0; q + 1 < kTeamMax; ++q)
          if (r == q && i >= static_cast<int>(n[q])) { i -= n[q]; ++r; }
      }
      key = TEAM ? ld_peer(cluster_map(smem_u32(list + i), min(r, team - 1))) : list[i];
      own = units(key);
      s.part_c[tid] = static_cast<int>(key);
      s.part_m[tid] = own;
    }
    __syncthreads();
    if (tid < ties) {
      int c = 0, same = 0;
      u64 m = 0;
#pragma unroll 4
      for (int j = 0; j < ties; ++j) {
        const uint32_t o = static_cast<uint32_t>(s.part_c[j]);
        const u64 w = s.part_m[j];
        if (o > key) { ++c; m += w; }
        same += o == key;
      }
      const bool last = c + same == ties;
      c += before_c;
      m += before_m;
      if (by_mass ? m < want && (last || want <= m + same * own) : static_cast<u64>(c) < want && (last || want <= static_cast<u64>(c + same))) {
        s.found_c = c; s.found_m = m; s.found_ties = same; s.found_at = static_cast<int>(key);
      }
    }
    __syncthreads();
    before_c = s.found_c; before_m = s.found_m; ties = s.found_ties;
    lo = hi = static_cast<uint32_t>(s.found_at);
  }
  // Divides what a search ended in until it is one value.
  __device__ void divide(bool by_mass, u64 want) {
    const int tid = threadIdx.x, lane = tid & 31;
    while (lo != hi) {
      if (ties <= kFew) return settle_few(by_mass, want);
      const int shift = max(0, 24 - __clz(hi - lo));
      u64* sub_m = s.sub_m[turn];
      int* sub_c = s.sub_c[turn];
      turn ^= 1;
      __syncthreads();
      for (int i = tid; i < 256; i += kVocabThreads) { sub_c[i] = 0; sub_m[i] = 0; }
      __syncthreads();
      row.template each<2>([&](const uint32_t (&u)[8], uint32_t ok) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = sort_key(u[j]);
          if (!(ok >> j & 1) || !is_more(u[j]) || k < lo || k > hi) continue;
          atomicAdd(&sub_c[(k - lo) >> shift], 1);
          add_shared(&sub_m[(k - lo) >> shift], units(k));
        }
      });
      meet();
      if (tid < 256) { s.part_c[tid] = at(sub_c, 255 - tid); s.part_m[tid] = at(sub_m, 255 - tid); }
      __syncthreads();
      if (tid < 32) {                            // eight parts a lane, then those of one lane
        int c = 0;
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { c += s.part_c[lane * 8 + i]; m += s.part_m[lane * 8 + i]; }
        settle(by_mass, want, c, m, before_c, before_m);
        const int l = s.found_at, c0 = s.found_c;
        const u64 m0 = s.found_m;
        __syncwarp();
        settle(by_mass, want, lane < 8 ? s.part_c[l * 8 + lane] : 0, lane < 8 ? s.part_m[l * 8 + lane] : 0ull, c0, m0);
        if (lane == 0) s.found_at += l * 8;
      }
      __syncthreads();
      before_c = s.found_c; before_m = s.found_m; ties = s.found_ties;
      const int part = 255 - s.found_at;
      lo += static_cast<uint32_t>(part) << shift;
      hi = min(hi, lo + ((1u << shift) - 1));
    }
  }
  // weight of the tokens that a search ended in, in units, and the mass of a prefix that ends there
  __device__ __forceinline__ double found_weight() const {
    if (many(bin)) return static_cast<double>(units(lo));
    return bin == kBins - 1 ? 0.0 : weight(value_of(bin)) * kUnit;
  }
  __device__ __forceinline__ u64 mass_of(int prefix) const { return before_m + static_cast<u64>(__double2ll_rn((prefix - before_c) * found_weight())); }

  __device__ __forceinline__ void clear() {
    uint4* t = reinterpret_cast<uint4*>(count - kCountAt);
    for (int i = threadIdx.x; i < kCountRoom / 4; i += kVocabThreads) t[i] = make_uint4(0, 0, 0, 0);
    if (F32) {
      t = reinterpret_cast<uint4*>(mass - kMassAt);
      for (int i = threadIdx.x; i < kMassRoom / 2; i += kVocabThreads) t[i] = make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_top[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kVocabWarps; ++w) v = max(v, s.warp_top[w]);
    return v;
  }
  __device__ __forceinline__ int block_sum(int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.sum_c[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kVocabWarps; ++w) v += s.sum_c[w];
    return v;
  }
  // The exponents that matter: up to the largest magnitude that a token of weight e^-44 or more can have.
  __device__ __forceinline__ int base_for(float top, double t) const {
    const double far = static_cast<double>(top) - 44.0 * t, most = isinf(top) ? 1e300 : fmax(fabs(static_cast<double>(top)), fabs(far));
    if (most >= 1.0 && most < 65536.0) return kUsualBase;
    const int e = most >= 3e38 ? (isinf(top) ? 128 : 127) : most < 1e-37 ? -126 : ilogb(most);
    return max(0, ((e - 47 + 127) << 7) - 1);
  }

  // One look at a bf16 row, two tokens in a word: places in the table with one clamped addition, one shift and one merge for both.  NaN and -inf
  // are counted with what is too large to have a bin.  Returns the largest value as a signed 16-bit number: the largest value if that is not negative.
  // `tiny`: whether the bin of zero holds another value of the thread's: the smallest magnitude less one, which takes zeros to the top.
  template <bool FILL>
  __device__ __forceinline__ int quick_look(bool& tiny) {
    constexpr uint32_t down = static_cast<uint32_t>(0x10000 - kUsualBase) * 0x10001u, limit = static_cast<uint32_t>(kSpan + 1) * 0x10001u;
    uint32_t top = 0x80008000u, least = 0xffffffffu;
    char* table = reinterpret_cast<char*>(count);
    auto places = [&](uint32_t w) {
      const uint32_t mag = w & 0x7fff7fffu;
      least = __viaddmin_u16x2(mag, 0xffffffffu, least);
      return (__viaddmin_s16x2_relu(mag, down, limit) << 2) | (w & 0x80008000u);
    };
    auto pair = [&](uint32_t w) {
      top = __vmaxs2(top, w);
      if (!FILL) return;
      const uint32_t place = places(w);
      atomicAdd(reinterpret_cast<int*>(table + (place & 0xffffu)), 1);
      atomicAdd(reinterpret_cast<int*>(table + (place >> 16)), 1);
    };
    auto some = [&](uint32_t w, uint32_t ok) {                               // two bits: which of the pair are allowed
      const uint32_t sel = (ok & 1 ? 0xffffu : 0u) | (ok & 2 ? 0xffff0000u : 0u);
      top = __vmaxs2(top, (w & sel) | (0x80008000u & ~sel));
      if (!FILL) return;
      const uint32_t place = places(w & sel);
      if (ok & 1) atomicAdd(reinterpret_cast<int*>(table + (place & 0xffffu)), 1);
      if (ok & 2) atomicAdd(reinterpret_cast<int*>(table + (place >> 16)), 1);
    };
    auto few = [&](const uint4& q, uint32_t ok) {                            // an allowed token at a time
      do {
        const int j = __ffs(ok) - 1;
        const uint32_t w = j & 4 ? (j & 2 ? q.w : q.z) : (j & 2 ? q.y : q.x), h = j & 1 ? w >> 16 : w & 0xffffu;
        top = __vmaxs2(top, h | 0x80000000u);
        if (FILL) atomicAdd(reinterpret_cast<int*>(table + (places(h) & 0xffffu)), 1);
        ok &= ok - 1;
      } while (ok);
    };
    const uint4* vec = reinterpret_cast<const uint4*>(row.base);
    const int tid = threadIdx.x, lane = tid & 31, first = row.from + (row.from < row.to && !row.whole(row.from)), last = row.to - (row.to > first && !row.whole(row.to - 1));
    const int tiles = (row.to - row.from + 31) >> 5;
    int most = -32768;
    constexpr int U = 4;
    for (int i0 = tid >> 5; i0 < tiles; i0 += U * kVocabWarps) {
      uint4 q[U];
      uint32_t ok[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {                  // values do not wait for their mask
        const int v = row.from + (i0 + k * kVocabWarps) * 32 + lane;
        const bool in = v >= first && v < last;
        if (in) q[k] = vec[v];
        ok[k] = in ? row.allowed(v) : 0u;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * kVocabWarps;
        if (i >= tiles) break;
        top = 0x80008000u;
        if (ok[k] == 0xffu) {
          pair(q[k].x); pair(q[k].y); pair(q[k].z); pair(q[k].w);
        } else if (ok[k] && __popc(ok[k]) <= 3) {
          few(q[k], ok[k]);
        } else if (ok[k]) {
          some(q[k].x, ok[k]); some(q[k].y, ok[k] >> 2); some(q[k].z, ok[k] >> 4); some(q[k].w, ok[k] >> 6);
        }
        const int t = __reduce_max_sync(0xffffffffu, max(static_cast<int>(top) >> 16, static_cast<int>(top << 16) >> 16));
        if (lane == 0) tile_max[i] = static_cast<short>(t);
        most = max(most, t);
      }
    }
    // the ends of the row: up to two vectors, a token a thread of the warp that has their tile
    for (int e = 0; e < 2; ++e) {
      const int end = e ? last : row.from, i = (end - row.from) >> 5;
      if ((e ? last == row.to : first == row.from) || i % kVocabWarps != tid >> 5) continue;
      int t = -32768;
      if (lane < 8 && row.first(end) + lane >= 0 && row.first(end) + lane < row.vocab && (row.allowed(end) >> lane & 1)) {
        const uint32_t h = reinterpret_cast<const unsigned short*>(row.base)[end * 8 + lane];
        if (FILL) {
          places(h);
          atomicAdd(&count[place_of(h << 16, kUsualBase)], 1);
        }
        t = static_cast<int>(static_cast<short>(h));
      }
      t = __reduce_max_sync(0xffffffffu, t);
      __syncwarp();
      if (lane == 0) tile_max[i] = static_cast<short>(max(t, static_cast<int>(tile_max[i])));
      most = max(most, t);
    }
    tiny = min(least & 0xffffu, least >> 16) < static_cast<uint32_t>(kUsualBase);
    return most;
  }
  // Any row: the largest key, and the table if FILL.
  template <bool FILL>
  __device__ __forceinline__ uint32_t look() {
    float top = -INFINITY;                       // NaN is no maximum
    row.template each<FILL ? (F32 ? 1 : 2) : kAhead>([&](const uint32_t (&u)[8], uint32_t ok) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = ok >> j & 1 ? __uint_as_float(u[j]) : -INFINITY;
        top = fmaxf(top, v);
        if (!FILL || !(v > -INFINITY)) continue;
        atomicAdd(&count[place_of(u[j], base)], 1);
        if (F32) add_shared(&mass[place_of(u[j], base)], units(sort_key(u[j])));
      }
    });
    return top > -INFINITY ? sort_key(__float_as_uint(top)) : 0u;
  }
};

template <bool F32, bool TEAM>
__global__ void __launch_bounds__(kThreadsOf<F32>, F32 ? 1 : 2)
sample_vocabulary_kernel(const CbVocabulary p, int team) {
  constexpr int kVocabThreads = kThreadsOf<F32>, kVocabWarps = kVocabThreads / 32;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ VocabScratch s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!TEAM) team = 1;
  const int rank = TEAM ? static_cast<int>(cluster_ctarank()) : 0, n_row = blockIdx.x / team;
  // the masses, the counts, the tiles
  u64* mass = reinterpret_cast<u64*>(dyn) + kMassAt;
  int* count = reinterpret_cast<int*>(dyn + (F32 ? kMassRoom * sizeof(u64) : 0)) + kCountAt;
  short* tile_max = reinterpret_cast<short*>(count - kCountAt + kCountRoom);
  pdl_wait();
  pdl_launch_dependents();
  const int r = p.rows_of ? p.rows_of[n_row] : n_row;
  if (r < 0 || r >= p.limit) return;
  const float temp = p.temperature ? p.temperature[r] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double t = greedy ? 1.0 : static_cast<double>(temp);
  Vocab<F32, TEAM> f{VocabRow<F32>(p, r, rank, team), s, count, mass, tile_max, rank, team, kUsualBase, false, 0ull, 0.f, 1.0 / t};
  f.turn = 0;
  if (tid == 0) s.owner = 0;
  if (!greedy) f.clear();
  f.meet();                                      // the peers run: their shared memory may be written

  // The largest value and, for a draw, the table.
  uint32_t best_key = 0;
  bool filled = false;
  if (!F32) {
    bool tiny = false;
    const int most = static_cast<int>(f.block_max(static_cast<uint32_t>((greedy ? f.template quick_look<false>(tiny) : f.template quick_look<true>(tiny)) + 32768))) - 32768;
    tiny = __syncthreads_or(tiny);
    // what the peers have to know: the largest, whether there are tiny values, tokens too large below zero (among them -inf and NaN)
    if (tid == 0) f.tell(s.told.top, static_cast<u64>(most + 32768) << 48 | static_cast<u64>(tiny) << 32 | (greedy ? 0ull : static_cast<u64>(count[kNegative + kSpan + 1])));
    f.meet();
    u64 top = 0, tinies = 0, low = 0;
    for (int c = 0; c < team; ++c) {
      const u64 v = s.told.top[c];
      top = max(top, v >> 48);
      tinies += v >> 32 & 1;
      low += v & 0xffffff;
    }
    const int value = static_cast<int>(top) - 32768;
    if (value >= 0 && value < 0x7f80 && low == 0) {
      best_key = sort_key(static_cast<uint32_t>(value) << 16);
      filled = greedy || f.base_for(key_value(best_key), t) == kUsualBase;
      f.mixed = tinies != 0;
    }
    if (!filled && !greedy) {
      f.meet();                                  // the peers may still read the table
      f.clear();
      f.mixed = false;
      __syncthreads();
    }
  }
  if (!filled) {
    // a look that knows what counts; in the usual bins at first, which most rows keep
    bool fill = !F32 && !greedy && best_key == 0;
    if (best_key == 0) {
      const uint32_t top = f.block_max(!F32 && fill ? f.template look<!F32>() : f.template look<false>());
      if (tid == 0) f.tell(s.told.zero_m, top);
      f.meet();
      for (int c = 0; c < team; ++c) best_key = max(best_key, static_cast<uint32_t>(s.told.zero_m[c]));
    }
    if (best_key == 0) {                         // nothing may be drawn
      if (tid == 0 && rank == 0) {
        p.ids[r] = 0;
        if (p.logprob) p.logprob[r] = -INFINITY;
        if (p.kept) p.kept[r] = 0;
      }
      if (TEAM) cluster_sync_all();              // a CTA's shared memory lives until the last word from its peers
      return;
    }
    if (!greedy) {
      f.best = key_value(best_key);
      const int base = f.base_for(f.best, t);
      if (!fill || base != kUsualBase) {
        f.meet();
        if (fill) { f.clear(); __syncthreads(); }
        f.base = base;
        f.template look<true>();
      }
      f.mixed = !F32;
      f.meet();
    }
  }
  f.best = key_value(best_key);

  uint32_t pick_key = best_key;
  int pick = 0;                                  // which of the tokens of that value, by id
  if (!greedy) {
    if (f.mixed && f.at(count, 0) + f.at(count, kNegative) == 0) f.mixed = false;
    if (f.mixed) {
      u64 m = 0;
      int other = 0;
      f.row.template each<2>([&](const uint32_t (&u)[8], uint32_t ok) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = place_of(u[j], f.base);
          if (!(ok >> j & 1) || !is_more(u[j]) || (d != 0 && d != kNegative)) continue;
          m += f.units(sort_key(u[j]));
          other |= (u[j] << 1) != 0;
        }
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      const int others = f.block_sum(other);
      if (lane == 0) s.sum_m[warp] = m;
      __syncthreads();
      m = 0;
      for (int w = 0; w < kVocabWarps; ++w) m += s.sum_m[w];
      f.meet();                                  // what is in the entries has been read
      if (tid == 0) { f.tell(s.told.zero_m, m); f.tell(s.told.least, static_cast<u64>(others)); }
      f.meet();
      f.zero_mass = f.told(s.told.zero_m);
      f.mixed = f.told(s.told.least) != 0;
      __syncthreads();
    }
    int total;
    u64 sum;
    f.sums(total, sum);
    int n = total;
    u64 kept = sum;
    const int k = p.top_k ? p.top_k[r] : 0;
    const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
    if (k > 0 && k < n) {
      f.find(false, k);
      n = k;
      kept = f.mass_of(n);
    }
    if (tp < 1.f) {
      const u64 want = max(1ull, static_cast<u64>(ceil(static_cast<double>(fmaxf(tp, 0.f)) * static_cast<double>(kept))));
      f.find(true, want);
      const double w = f.found_weight();
      const int m = min(f.ties, max(1, static_cast<int>(ceil(static_cast<double>(want - f.before_m) / w))));
      if (f.before_c + m < n) {
        n = f.before_c + m;
        kept = f.mass_of(n);
      }
    }
    if (mp >= kLeastMinP) {
      const double least = fmin(static_cast<double>(mp), 1.0);
      int c = 0;
      if (F32 || f.mixed) {
        // most tokens are told by one comparison with a little less than the smallest value that is heavy enough
        const double far = log(least), edge = f.best + far * t;
        const float cut = isfinite(edge) ? static_cast<float>(edge - 1e-5 * (fabs(static_cast<double>(f.best)) + fabs(far * t)) - 1e-37) : f.best == INFINITY ? INFINITY : -INFINITY;
        f.row.template each<f.kAhead>([&](const uint32_t (&u)[8], uint32_t ok) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((ok >> j & 1) && __uint_as_float(u[j]) >= cut) c += f.heavy_one(__uint_as_float(u[j]), far);
        });
        c = f.block_sum(c);
        f.meet();
        if (tid == 0) f.tell(s.told.least, static_cast<u64>(c));
        f.meet();
        c = static_cast<int>(f.told(s.told.least));
      } else {
        c = f.heavy(least);
      }
      c = max(1, c);
      if (c < n) {
        n = c;
        f.find(false, n);
        kept = f.mass_of(n);
      }
    }
    float u = p.uniforms ? p.uniforms[r] : philox_uniform(p.seeds ? p.seeds[r] : 0ull, p.counters ? p.counters[r] : 0ull);
    u = fminf(fmaxf(u, 0.f), 0.99999994f);
    const double aim = static_cast<double>(u) * static_cast<double>(kept);
    f.find(true, static_cast<u64>(aim) + 1);
    const double w = f.found_weight();
    pick = w > 0.0 ? static_cast<int>((aim - static_cast<double>(f.before_m)) / w) : 0;
    pick = max(0, min(pick, min(f.ties, n - f.before_c) - 1));
    pick_key = f.many(f.bin) ? f.lo : f.value_of(f.bin);
    if (tid == 0 && rank == 0) {
      const float v = key_value(pick_key);
      if (p.logprob) p.logprob[r] = static_cast<float>((v == f.best ? 0.0 : (static_cast<double>(v) - f.best) * f.inv_t) - log(static_cast<double>(kept) / kUnit));
      if (p.kept) p.kept[r] = n;
    }
  } else if (tid == 0 && rank == 0) {
    if (p.logprob) p.logprob[r] = 0.f;
    if (p.kept) p.kept[r] = 1;
  }

  // the token: how many of the value are in every tile of 256, then a look at the tile that holds it
  f.meet();                                      // the peers read the table no more
  const int tiles = (f.row.to - f.row.from + 31) >> 5;
  unsigned short* in_tile = reinterpret_cast<unsigned short*>(dyn);
  const float pick_value = key_value(pick_key);
  // of a positive bf16 value only the tiles whose largest is no less
  const bool some = !F32 && pick_value > 0.f;
  const int least = static_cast<int>(__float_as_uint(pick_value) >> 16);
  const bool plain = !F32 && !f.row.mask && pick_value != 0.f;
  const uint32_t twice = (__float_as_uint(pick_value) >> 16) * 0x10001u;
  auto of_tile = [&](int v, uint32_t ok, const uint4& a, const uint4& b) {
    if (ok == 0) return 0;
    if (plain && f.row.whole(v)) return (__popc(__vcmpeq2(a.x, twice)) + __popc(__vcmpeq2(a.y, twice)) + __popc(__vcmpeq2(a.z, twice)) + __popc(__vcmpeq2(a.w, twice))) >> 4;
    uint32_t u[8];
    ok = f.row.values(v, ok, a, b, u);
    int c = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) c += (ok >> j & 1) && __uint_as_float(u[j]) == pick_value;       // zeros are one
    return c;
  };
  int found = 0;
  for (int i0 = warp; i0 < tiles; i0 += 32 * kVocabWarps) {                   // a tile a lane to begin with
    const int mine = i0 + lane * kVocabWarps;
    if (mine < tiles) in_tile[mine] = 0;
    uint32_t todo = __ballot_sync(0xffffffffu, mine < tiles && (!some || f.tile_max[mine] >= least));
    __syncwarp();
    while (todo) {
      constexpr int U = f.kAhead;
      int i[U], c[U];
      uint32_t ok[U];
      uint4 a[U], b[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        i[k] = todo ? i0 + (__ffs(todo) - 1) * kVocabWarps : -1;
        todo &= todo - 1;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int v = f.row.from + i[k] * 32 + lane;
        const bool in = i[k] >= 0 && v < f.row.to;
        f.row.fetch(v, in, a[k], b[k]);
        ok[k] = in ? f.row.allowed(v) : 0u;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) c[k] = of_tile(f.row.from + i[k] * 32 + lane, ok[k], a[k], b[k]);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (!__any_sync(0xffffffffu, c[k])) continue;
        const int n = __reduce_add_sync(0xffffffffu, c[k]);
        if (lane == 0) in_tile[i[k]] = static_cast<unsigned short>(n);
        found += n;
      }
    }
  }
  if (TEAM) {
    found = f.block_sum(lane == 0 ? found : 0);
    if (tid == 0) f.tell(s.told.ids, static_cast<u64>(found));
    f.meet();                                    // the last word between the CTAs
    for (int c = 0; c < rank; ++c) pick -= static_cast<int>(s.told.ids[c]);
    if (pick < 0 || pick >= found) return;
  } else {
    __syncthreads();
  }
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
  const int v = f.row.from + tile * 32 + lane;
  uint32_t hit = 0;
  if (v < f.row.to) {
    uint32_t u[8], ok = f.row.allowed(v);
    uint4 a, b;
    f.row.fetch(v, true, a, b);
    ok = f.row.values(v, ok, a, b, u);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((ok >> j & 1) && __uint_as_float(u[j]) == pick_value) hit |= 1u << j;
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
    p.ids[r] = f.row.first(v) + __ffs(hit) - 1;
  }
}

template <bool F32, bool TEAM>
static cudaError_t vocabulary_launch(const CbVocabulary& p, int team, cudaStream_t stream) {
  const int smem = kCountRoom * 4 + (F32 ? kMassRoom * 8 : (p.vocab / (256 * team) + 3) * 2);
  static int ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || ready[dev] < smem) {
    e = cudaFuncSetAttribute(sample_vocabulary_kernel<F32, TEAM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev] = smem;
  }
  return launch(sample_vocabulary_kernel<F32, TEAM>, dim3(p.rows * team), dim3(kThreadsOf<F32>), smem, stream, dim3(team, 1, 1), p, team);
}

}  // namespace cb

extern "C" int cb_sample_vocabulary(const CbVocabulary* p, void* stream) {
  using namespace cb;
  if (p->rows < 0 || p->vocab < 1 || p->vocab > kVocabMax || p->ld < p->vocab || (p->mask && p->ld_mask < 0)) return -10;
  if (reinterpret_cast<uintptr_t>(p->logits) % (p->f32 ? 4 : 2)) return -11;
  if (p->rows == 0) return 0;
  // CTAs of a row: as many as find an SM each, with work for each.  bf16 rows of 151936 tokens with top-k, limit 296 -> 148: 20 rows 21.5 -> 18.7 us,
  // 48 23.8 -> 22.4, 74 38 -> 22.6 (clusters that do not fit at once), 100 30.8 -> 25.6.  (Other vocabularies were not measured.)
  int team = 1;
  while (team < kTeamMax && static_cast<long long>(p->rows) * team * 2 <= 148 && p->vocab / (team * 2) >= 4096) team *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->f32 ? (team > 1 ? vocabulary_launch<true, true>(*p, team, st) : vocabulary_launch<true, false>(*p, 1, st))
                               : (team > 1 ? vocabulary_launch<false, true>(*p, team, st) : vocabulary_launch<false, false>(*p, 1, st));
  return static_cast<int>(e);
}
