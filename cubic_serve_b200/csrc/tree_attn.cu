// Attention of trees of drafted tokens over the paged quantised cache (page layout: kv_layout.cuh).
//
// Request i has start[i] tokens in the cache and count[i] nodes behind them, at the slots start[i] + j in the order of the nodes.  Node j is row
// row0[i] + j of q and out; it sees the whole context and those nodes j' whose bit is set in its row of `masks`:
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  t over what the row sees; zeros where that is nothing.
// A cached value is a code times an fp32 scale, one per token and 32 channels.
#include "paged_attn.cuh"

// Packed by ops/native.py::TREE_ATTN.
struct CbTreeAttn {
  const __nv_bfloat16* q;    // [rows, Hq * 128], row stride ldq
  __nv_bfloat16* out;        // likewise, ldo
  const uint8_t* cache;      // [pages][Hkv][blob]
  const int* table;          // [table_rows, width], row stride ld
  const int* request;        // [n] row of the block table
  const int* row0;           // [n] first row of the request
  const int* count;          // [n] nodes
  const int* start;          // [n] tokens of the context
  const uint32_t* masks;     // [rows, words], row stride ldm
  uint32_t* status;
  float* partial;            // cb_tree_attn_floats of them
  long long ldq, ldo, ld, ldm;
  int n, rows, table_rows, width, pages, words;
  int Hq, Hkv, k_bits, v_bits;
  float scale;
};

namespace cb {

static constexpr int kTreeMaxRequests = 1024, kTreeMaxWords = 8, kTreeMaxGroup = 128;

// What a launch is told of a request, checked: nodes that do not fit their rows or their masks, and contexts that the block table has no room for, see nothing.
struct TreeRequest {
  int slot, row0, count, start, total;   // count: rows to write; total: tokens to look at, 0: write zeros
};
__device__ __forceinline__ TreeRequest tree_request(const CbTreeAttn& p, int i, bool& bad) {
  TreeRequest r;
  r.slot = p.request[i];
  r.row0 = p.row0[i];
  r.count = p.count[i];
  r.start = p.start[i];
  if (r.count <= 0 || r.row0 < 0 || r.count > p.rows - r.row0) {
    bad = bad || r.count != 0;
    r.count = r.total = 0;
    return r;
  }
  const bool fits = r.slot >= 0 && r.slot < p.table_rows && r.count <= 32 * p.words && r.start >= 0 && r.start <= p.width * kPageTokens - r.count;
  bad = bad || !fits;
  r.total = fits ? r.start + r.count : 0;
  return r;
}
__device__ __forceinline__ int tree_page(const CbTreeAttn& p, int slot, int i, bool& bad) {
  const int page = p.table[slot * p.ld + i];
  const bool there = page >= 0 && page < p.pages;
  bad = bad || !there;
  return there ? page : 0;
}

// The page layout as constants (kv_layout.cuh)
template <int KBITS, int VBITS>
struct TreeLay {
  static constexpr int kScale = kPageTokens * kD * KBITS / 8, kBytesOfScales = kPageTokens * (kD / kKvGroup) * 4, vCode = kScale + kBytesOfScales,
                       vScale = vCode + kPageTokens * kD * VBITS / 8, bytes = vScale + kBytesOfScales, stride = (bytes + 127) & ~127;
};

// One row over the tokens [lo, hi) in fp32, by a warp whose lanes have four channels each.  `sees`: the row's words.
template <int KBITS, int VBITS>
__device__ __forceinline__ void tree_row(const CbTreeAttn& p, const TreeRequest& r, int kvh, int lo, int hi, const uint32_t* sees, const __nv_bfloat16* q,
                                         int lane, float& m, float& sum, float (&o)[4], bool& bad) {
  using L = TreeLay<KBITS, VBITS>;
  constexpr float kBias = 1 << (KBITS - 1), vBias = 1 << (VBITS - 1);
  const uint2 qw = reinterpret_cast<const uint2*>(q)[lane];
  const float2 q01 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qw.x)), q23 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qw.y));
  const float qf[4] = {q01.x, q01.y, q23.x, q23.y}, scale = p.scale * 1.4426950408889634f;
  m = -INFINITY;
  sum = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] = 0.f;
#pragma unroll 1
  for (int t = lo; t < hi; ++t) {
    const int j = t - r.start;
    if (j >= 0 && !(sees[j >> 5] >> (j & 31) & 1u)) continue;
    const int page = tree_page(p, r.slot, t / kPageTokens, bad), tok = t % kPageTokens;
    const uint8_t* blob = p.cache + (static_cast<size_t>(page) * p.Hkv + kvh) * L::bytes;
    const uint32_t kc = pf_codes_k<KBITS>(blob, tok, lane), vc = pf_codes_v<VBITS>(blob + L::vCode, tok, lane);
    const float ks = *reinterpret_cast<const float*>(blob + L::kScale + tok * 16 + (lane >> 3) * 4);
    const float vs = *reinterpret_cast<const float*>(blob + L::vScale + tok * 16 + (lane >> 3) * 4);
    float z = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) z = fmaf(qf[c], (static_cast<float>(kc >> (8 * c) & 255u) - kBias) * ks, z);
    z = warp_sum(z) * scale;
    if (z > m) {
      const float alpha = fast_exp2(m - z);
      m = z;
      sum *= alpha;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] *= alpha;
    }
    const float pr = fast_exp2(z - (m == -INFINITY ? 0.f : m));
    sum += pr;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = fmaf(pr, (static_cast<float>(vc >> (8 * c) & 255u) - vBias) * vs, o[c]);
  }
}

// ------------------------------------------------------------------------------------------------- schedule
// An item is up to 256 rows (node x query head of the group) of a request and key / value head, in steps of 64 tokens.  The slots of all items, one after the
// other, are dealt out evenly: CTA c takes those that begin at the units [c per, (c + 1) per), however uneven the requests are.  An item has a slot for each step, and
// kTrSwitch before them: its queries and its results take as long as five steps (dealt out by steps alone 32 x 64 behind up to 1500 took 142 us in place of 121, 2 x 64
// behind 32000 122 in place of 113).  An item that several CTAs share leaves a part (its maximum, sum and unnormalised output) of each in the workspace, and
// tree_merge_kernel joins them in order: no atomics, the same bits every time.
static constexpr int kTrTiles = 2, kTrRows = 128, kTrItemRows = kTrTiles * kTrRows;
static constexpr int kTrPages = 4, kTrTok = kTrPages * kPageTokens;
static constexpr int kTrThreads = 640;
// Registers go to the softmax, whose loops keep a row's scores (64 x 16 behind 4096: with 128 of them 265 us, 136: 252, 144: 245), as long as the warps of the second line
// spill nothing in their loops (32 x 64 with 56 and 48 for these: 127 us in place of 121).
static constexpr int kTrRegs = 96, kTrRegsSoftmax = 144, kTrRegsConvert = 64, kTrRegsOther = 64;
static_assert(2 * kTrRegsSoftmax + 2 * kTrRegsConvert + kTrRegsOther <= 5 * kTrRegs, "five warpgroups");
static constexpr int kTrLists = 4, kTrRaw = 4;
// Operands: of K of two steps, of V, which waits longer, of four.  A step's places, the four warps that convert it and, of items in both tiles, its tile go by its number in
// the CTA, so that whoever waits at a place has waited for each of its steps before.
static constexpr int kTrOpsK = 2, kTrOpsV = 4;
// Steps whose powers of two are kept: the note of step s is written behind raw_full (s) <- raw_free (s - kTrRaw) <- v_free of step s - kTrRaw - kTrOpsV <- p_full of the
// tiles that take part in it, which have read theirs by then.
static constexpr int kTrNotes = 8;
static_assert(kTrRaw % 2 == 0 && kTrNotes % 2 == 0 && kTrRaw + kTrOpsV <= kTrNotes, "even and odd steps have their own places");
static constexpr int kTrSwitch = 5;                      // slots that an item takes in the schedule before its steps
static constexpr float kTrGrowth = 2.f;
static constexpr int kTrApart = 9;                       // powers of two that scales are apart: up to here the short conversion, ...
static constexpr int kTrApartK = 18, kTrApartV = 14;     // ... and the long one
static constexpr int kTrHalf = kTrTok * 128;             // bytes of 64 channels of a step
static constexpr uint32_t kTrTmemCols = 512, kTrTmemTile = 256, kTrTmemP = 64, kTrTmemQ = 96, kTrTmemO = 128;

// Waits of a launch are bounded by `limit`: a warp's 32 rows of the fp32 program take 720 cycles a row and token (pages in the L2 cache), behind 130000 tokens longer than other kernels' waits
// may, so that the longest context there can be counts in it (tr_limit).  What follows a wait that is not over at once is out of the way of the loops.
__device__ __forceinline__ bool tr_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, long long limit) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
  return mbar_wait_park(bar, parity, abort_flag, limit);
}
static constexpr long long kTrSlowCycles = 4096;         // of a row and token, with room to spare
static inline long long tr_limit(const CbTreeAttn& p) { return kWaitBudgetCycles + 32 * kTrSlowCycles * kPageTokens * p.width; }
// Where a role stands in a ring of n places, and the parity that it waits for there
struct TrRing {
  int i, n;
  uint32_t phase;
  __device__ __forceinline__ explicit TrRing(int places, uint32_t parity = 0, int at = 0) : i(at), n(places), phase(parity) {}
  __device__ __forceinline__ void advance(int by = 1) {
    i += by;
    if (i >= n) { i -= n; phase ^= 1u; }
  }
};
struct TrItem {
  int kvh;                                               // < 0: no more items
  int slot, row0, count, start, total;                   // the request
  int first, rows;                                       // rows [first, first + rows) of its count x group
  int lo, steps;                                         // steps [lo, lo + steps) of this CTA; none: zeros
  int part;                                              // place of its part, -1: the whole item
};
struct TrDesc { int parts, row0, first, rows, kvh, pad[3]; };
struct __align__(1024) TrSmem {
  uint8_t q[kTrTiles][kTrRows * 128];                    // f16, channels 64..127: [row][128 B], 16-byte chunk ^ (row & 7)
  uint8_t k[kTrOpsK][2 * kTrHalf];                             // f16 [stage][64-channel half][token][128 B]
  uint8_t v[kTrOpsV][2 * kTrHalf];                             // likewise
  struct Note {
    float k, v;                                          // of a step: what the scales of K and V are multiplied with, ...
    int k_wide, v_wide;                                  // ... and whether the long conversion takes them
    float back;                                          // scores are this times what the MMAs give
    int v_exp;                                           // output is 2^v_exp times ...
  } note[kTrNotes];
  uint32_t redo[kTrLists];                               // of an item's steps: some values are beyond what f16 operands hold
  uint64_t raw_full[kTrRaw], raw_free[kTrRaw], k_full[kTrTiles][kTrOpsK], k_free[kTrOpsK], v_full[kTrTiles][kTrOpsV], v_free[kTrOpsV], note_full[kTrNotes];
  uint64_t list_full[kTrLists], list_free[kTrLists], q_full[kTrTiles], s_full[kTrTiles], s_free[kTrTiles], p_full[kTrTiles], pv_done[kTrTiles];
  uint64_t exch_full, exch_free;
  TrItem list[kTrLists];
  float2 exch_ml[kTrTiles][kTrRows];                     // rows in both tiles: maximum and sum, ...
  int exch_exp[kTrTiles][kTrRows];                       // ... and v_exp
  uint32_t tmem, abort_word;
  long long upto[kTreeMaxRequests + 1], items[kTreeMaxRequests + 1];     // units of the requests before; their items' units a slot
};

// Items of one tile's rows have them in both tiles, which take its steps in turn (two warps of a kind on a scheduler where one would wait for itself).
__device__ __forceinline__ bool tr_split(const TrItem& l) { return l.rows <= kTrRows; }
// The first step of an item that tile t takes; `before`: steps of the CTA before the item.
__device__ __forceinline__ int tr_first(const TrItem& l, int t, int before) { return tr_split(l) ? (before ^ t) & 1 : 0; }

__device__ __forceinline__ long long tr_divide(long long a, long long b) {       // (most numbers have 32 bits)
  return (a | b) >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}
__device__ __forceinline__ int tr_steps(const TreeRequest& r) { return max(1, (r.total + kTrTok - 1) / kTrTok); }
// Units of the schedule that a step takes: one if its request's items are in both tiles (tr_split), else two.
__device__ __forceinline__ int tr_slot(const TreeRequest& r, int G) { return r.count * G <= kTrRows ? 1 : 2; }
__device__ __forceinline__ int tr_groups(const TreeRequest& r, int G) { return (r.count * G + kTrItemRows - 1) / kTrItemRows; }
static inline int tr_rows(int words, int rows, int G) {
  const long long most = static_cast<long long>(words * 32 < rows ? words * 32 : rows) * G;
  return most < kTrItemRows ? static_cast<int>(most) : kTrItemRows;
}

// One step's codes into operands: code times scale, in f16.  A byte b (the code and its bias) in the low bits of an f16 is the number 2^-24 b, exactly.
// Short: with the scale as f16 times 2^24 that takes one multiply-add, b S - bias S, of two roundings (the scale's and the product's, 2^-11 each), as long as what the
// operands hold is below 2^-2 and their scales are no more than 2^9 apart: below 2^-14 f16 has steps of 2^-24.
// WIDE: the code as f16 (a subtraction) times sh + sl, f16 each: the product with sl, rounded, is 2^-11 of the whole, so that the multiply-add behind it rounds once
// what 32-bit arithmetic would; values up to 2^15.
// So keys and values have 10 to 11 bits here, where the prompt kernel keeps pairs of f16 (20 and 18); probabilities are f16 in both, their sum takes them in 32 bits.  On
// caches as servers fill them the result's own rounding to bf16 is 1.66e-3 of it; what comes before adds 0.75 to 0.9e-3 with the short conversion, 0.46 to 0.6e-3 with the
// long one throughout, which takes longer (64 x 16 behind 4096 279 us in place of 242, 32 x 64 128 for 122, 2 x 64 behind 32000 103 for 99), pairs of f16 twice the products.
// What K holds of tokens that no row sees is masked with their scores.
__device__ __forceinline__ void tr_put(uint32_t to, const uint4& x) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
__device__ __forceinline__ uint32_t tr_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t tr_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// the two numbers that a scale times the step's power of two is taken as
template <int BITS, bool WIDE>
__device__ __forceinline__ void tr_scale(float s, uint32_t& a, uint32_t& b) {
  if constexpr (WIDE) {
    pf_split(s, a, b);
  } else {
    constexpr uint32_t bias = BITS == 8 ? 0x80808080u : BITS == 6 ? 0x80208020u : 0x80088008u;           // -bias 2^-24
    a = pack_f16x2(s, s);
    b = tr_mul(a, bias);
  }
}
// the bytes that `sel` takes of a word
template <int BITS, bool WIDE>
__device__ __forceinline__ uint32_t tr_pair(uint32_t word, uint32_t sel, uint32_t a, uint32_t b) {
  if constexpr (WIDE) {
    const uint32_t code = u8x2_to_f16x2(word, sel, BITS == 8 ? 0x64806480u : BITS == 6 ? 0x64206420u : 0x64086408u);
    return tr_fma(code, a, tr_mul(code, b));
  } else {
    return tr_fma(prmt(word, 0u, sel), a, b);
  }
}
template <int BITS, bool WIDE>
__device__ __forceinline__ uint4 tr_eight(uint32_t x, uint32_t y, uint32_t a, uint32_t b) {              // eight bytes in order
  return make_uint4(tr_pair<BITS, WIDE>(x, 0x5140u, a, b), tr_pair<BITS, WIDE>(x, 0x5342u, a, b), tr_pair<BITS, WIDE>(y, 0x5140u, a, b), tr_pair<BITS, WIDE>(y, 0x5342u, a, b));
}
// (The loops stay loops: five kinds of warps run their code at the same time, and unrolled it does not fit the instruction caches: 3700 cycles a step.)
template <int KBITS, int VBITS, bool WIDE>
__device__ __forceinline__ void tr_convert_k(uint8_t* k, const uint8_t* raw, float mul, int tid) {
  using L = TreeLay<KBITS, VBITS>;
  // an item is a scale's 32 channels of a token
  const int tok = tid & 15, g = tid >> 4 & 3, sw = tok & 7;
  raw += (tid >> 6) * L::stride;
  const uint8_t* codes = raw + tok * 16 + g * (KBITS == 8 ? 512 : 256);
  const uint8_t* high = raw + kPageTokens * kD / 2 + g * 128 + (tok & 7) * 16;
  const uint8_t* scale = raw + L::kScale + tok * 16 + g * 4;
  // chunks 4 (g & 1) + {0, 1, 2, 3} of the token's row, each ^ (row & 7)
  k += (g >> 1) * kTrHalf + ((tid >> 6) * 16 + tok) * 128 + (((g & 1) * 4 ^ (sw & 6)) << 4);
  const int one = (sw & 1) << 4;
#pragma unroll 1
  for (int page = 0; page < kTrPages / 2; ++page) {
    uint32_t sh, sl;
    tr_scale<KBITS, WIDE>(*reinterpret_cast<const float*>(scale) * mul, sh, sl);
    uint4 x, w = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (KBITS != 8) x = *reinterpret_cast<const uint4*>(codes);
    if constexpr (KBITS == 6) {
      w = *reinterpret_cast<const uint4*>(high);
      if (tok >= 8) { w.x <<= 4; w.y <<= 4; w.z <<= 4; w.w <<= 4; }                      // (what leaves a byte's bits 4 to 7 is masked)
    }
    uint32_t to = smem_u32(k);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {                        // 16 channels
      uint4 n;
      if constexpr (KBITS == 8) {
        n = *reinterpret_cast<const uint4*>(codes + h * 256);
      } else {
        n = make_uint4(x.x & 0x0F0F0F0Fu, x.y & 0x0F0F0F0Fu, x.z & 0x0F0F0F0Fu, x.w & 0x0F0F0F0Fu);
        x = make_uint4(x.x >> 4, x.y >> 4, x.z >> 4, x.w >> 4);
        if constexpr (KBITS == 6) {
          n = make_uint4(n.x | (w.x & 0x30303030u), n.y | (w.y & 0x30303030u), n.z | (w.z & 0x30303030u), n.w | (w.w & 0x30303030u));
          w = make_uint4(w.x >> 2, w.y >> 2, w.z >> 2, w.w >> 2);
        }
      }
      tr_put(to + one, tr_eight<KBITS, WIDE>(n.x, n.y, sh, sl));
      tr_put(to + (one ^ 16), tr_eight<KBITS, WIDE>(n.z, n.w, sh, sl));
      to ^= 32;
    }
    codes += 2 * L::stride; high += 2 * L::stride; scale += 2 * L::stride;
    k += 2 * 16 * 128;
  }
}
// V from `visible` on becomes zeros: those slots may hold anything, and a probability of zero has to stay zero.
template <int KBITS, int VBITS, bool WIDE>
__device__ __forceinline__ void tr_convert_v(uint8_t* v, const uint8_t* raw, int visible, float mul, int tid) {
  using L = TreeLay<KBITS, VBITS>;
  // an item is 16 channels of a token pair, eight at a time: lanes 0-3 of eight take the first eight first, the others the second (no bank twice)
  const int c = tid & 7, pair = tid >> 3 & 7, first = tid >> 2 & 1;
  const int at = (4 * c) ^ ((pair & 3) << 2);
  raw += (tid >> 6) * L::stride;
  const uint8_t* codes = raw + L::vCode + (VBITS == 8 ? pair * 256 + at * 8 : pair * 128 + at * 4);
  const uint8_t* high = raw + L::vCode + kPageTokens * kD / 2 + (pair & 3) * 128 + at * 4;
  const uint8_t* scale = raw + L::vScale + pair * 32 + (c >> 1) * 4;
  // chunk 2 c + half of rows 2 pair and 2 pair + 1, each ^ (row & 7)
  v += (c >> 2) * kTrHalf + ((tid >> 6) * 16 + pair * 2) * 128 + ((((2 * c) & 7) ^ ((pair & 3) * 2)) << 4);
  int tok = (tid >> 6) * 16 + pair * 2;
#pragma unroll 1
  for (int page = 0; page < kTrPages / 2; ++page, tok += 32) {
    uint32_t sh[2], sl[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f = *reinterpret_cast<const float*>(scale + h * 16) * mul;
      if (tok + h >= visible || !(fabsf(f) < INFINITY)) f = 0.f;
      tr_scale<VBITS, WIDE>(f, sh[h], sl[h]);
    }
    const uint32_t to = smem_u32(v);
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      const int half = first ^ e;
      uint4 x;
      if constexpr (VBITS == 8) {
        x = *reinterpret_cast<const uint4*>(codes + half * 16);
      } else {
        const uint2 n = *reinterpret_cast<const uint2*>(codes + half * 8);
        uint2 hw = make_uint2(0u, 0u);
        if constexpr (VBITS == 6) {
          hw = *reinterpret_cast<const uint2*>(high + half * 8);
          const int up = pair < 4 ? 0 : 4;
          hw.x <<= up; hw.y <<= up;
        }
        x = make_uint4(n.x, n.y, hw.x, hw.y);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 f;
        if constexpr (VBITS == 8) {
          const uint32_t sel = h ? 0x5341u : 0x5240u;
          f = make_uint4(tr_pair<8, WIDE>(x.x, sel, sh[h], sl[h]), tr_pair<8, WIDE>(x.y, sel, sh[h], sl[h]), tr_pair<8, WIDE>(x.z, sel, sh[h], sl[h]), tr_pair<8, WIDE>(x.w, sel, sh[h], sl[h]));
        } else {
          uint2 n = h ? make_uint2((x.x >> 4) & 0x0F0F0F0Fu, (x.y >> 4) & 0x0F0F0F0Fu) : make_uint2(x.x & 0x0F0F0F0Fu, x.y & 0x0F0F0F0Fu);
          if constexpr (VBITS == 6) {
            n.x |= (h ? x.z >> 2 : x.z) & 0x30303030u;
            n.y |= (h ? x.w >> 2 : x.w) & 0x30303030u;
          }
          f = tr_eight<VBITS, WIDE>(n.x, n.y, sh[h], sl[h]);
        }
        tr_put(to + h * 128 + ((half ^ h) << 4), f);
      }
    }
    codes += 2 * L::stride; high += 2 * L::stride; scale += 2 * L::stride;
    v += 2 * 16 * 128;
  }
}
// The smallest magnitude of a token's scales that is not zero, as bits
__device__ __forceinline__ uint32_t tr_least(const float4& s) {
  auto magnitude = [](float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b == 0u ? 0x7F800000u : b;
  };
  return min(min(magnitude(s.x), magnitude(s.y)), min(magnitude(s.z), magnitude(s.w)));
}

__device__ __forceinline__ void tr_tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tr_tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
}

// 64 bits: which of the tokens [tok0, tok0 + 64) a row sees.  `sees`: its words.
__device__ __forceinline__ uint2 tr_visible(const uint32_t* sees, int words, int start, int total, int tok0) {
  auto word = [&](int k) { return k >= 0 && k < words ? sees[k] : 0u; };
  const int j0 = tok0 - start, w = j0 >> 5, b = j0 & 31;               // (rounded down: the bits before node 0 are the context's)
  const uint32_t w0 = word(w), w1 = word(w + 1), w2 = word(w + 2);
  uint2 m = make_uint2(__funnelshift_r(w0, w1, b), __funnelshift_r(w1, w2, b));
  if (j0 < 0) {
    m.x |= -j0 >= 32 ? ~0u : (1u << -j0) - 1u;
    if (j0 < -32) m.y |= -j0 >= 64 ? ~0u : (1u << (-j0 - 32)) - 1u;
  }
  const int n = total - tok0;
  if (n < 64) m.y &= n <= 32 ? 0u : (1u << (n - 32)) - 1u;
  if (n < 32) m.x &= (1u << max(n, 0)) - 1u;
  return m;
}

// Roles: warps 0-7 own a row a thread (softmax needs no exchange: tensor-memory lane = row); warps 8-11 convert raw pages to the swizzled operands of K
// and V ([token][channel], f16), by turns with warps 12-15; warps 16 and 18 issue the MMAs of a tile each; warp 17 makes the items and copies pages;
// warp 19 finds the powers of two that bring a step's values into f16's range.
// Tensor memory of a tile of 128 rows: scores, probabilities (the A operand of their product), output and the first half of Q's channels; the other half of
// Q is in shared memory.  The scores of step i + 1 are computed while the softmax of step i runs.  The output is rescaled only when a row's maximum has grown by more
// than a factor of four: until then probabilities relative to the older maximum are at most 4.
// Powers of two keep operands in the range of f16: a row's for Q (undone with the softmax' scale: its 8 bits stay exact), a step's for K (likewise), one for V that grows
// with the largest scale (undone with the output).  Items whose scales are further apart than that holds (2^18 in a step of K, 2^14 in a CTA's steps of V), or not finite,
// are computed in fp32 (tree_row), a row at a time, 370 ns a token: a hundred times as long.  A group of zeros is stored with a scale of one, so that one of them among values
// whose scales are below 2^-14 is enough for that.
// Nothing is full: issue slots are half taken (16384 scores and as many codes a step of 256 rows, five warps a scheduler), matrix units for a quarter of the time, memory for as much.
// What a step waits for is its own chain from role to role, and instructions: warps whose rows a narrow tree does not have run the softmax all the same, items of one
// request convert the same pages anew, programs that differ share the instruction caches (any role's loops unrolled: 3 to 11 % slower; six more behind every wait: 9 %).
// 64 x 16 behind 4096 (8 bits, 32 / 8 heads) 242 us, 2.6 TB/s of the cache; 2 x 64 behind 32000 (K 4 bits, 32 / 4) 100 us; 32 x 64 behind up to 1500 (6 bits, 64 / 4) 122 us.
// One request of 8 nodes behind 700 tokens is a chain of latencies: 15 us, of which the second launch is 4.
// Every wait is bounded; on a timeout the roles leave, the status word is set and tensor memory is freed.
template <int KBITS, int VBITS>
__global__ void __launch_bounds__(kTrThreads, 1)
tree_kernel(const CbTreeAttn p, const int part_rows, const long long limit) {
  using L = TreeLay<KBITS, VBITS>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  TrSmem& sm = *reinterpret_cast<TrSmem*>(smem_raw + (-smem_u32(smem_raw) & 1023u));      // (by way of an integer it would be a generic address)
  uint8_t* raw = reinterpret_cast<uint8_t*>(&sm + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.Hq / p.Hkv;
  volatile uint32_t* abort_flag = &sm.abort_word;
  float* part_o = p.partial;
  float2* part_ml = reinterpret_cast<float2*>(part_o + static_cast<size_t>(gridDim.x) * 2 * part_rows * kD);
  TrDesc* desc = reinterpret_cast<TrDesc*>(part_ml + static_cast<size_t>(gridDim.x) * 2 * part_rows);
  if (tid == 0) {
    for (int b = 0; b < kTrRaw; ++b) {
      mbar_init(smem_u32(&sm.raw_full[b]), 1);
      mbar_init(smem_u32(&sm.raw_free[b]), 4);
    }
    for (int b = 0; b < kTrOpsV; ++b) {
      if (b < kTrOpsK) mbar_init(smem_u32(&sm.k_free[b]), 2);            // an MMA warp each, or one of them twice
      mbar_init(smem_u32(&sm.v_free[b]), 2);
      for (int t = 0; t < kTrTiles; ++t) {
        if (b < kTrOpsK) mbar_init(smem_u32(&sm.k_full[t][b]), 4);
        mbar_init(smem_u32(&sm.v_full[t][b]), 4);
      }
    }
    for (int b = 0; b < kTrNotes; ++b) {
      mbar_init(smem_u32(&sm.note_full[b]), 1);
    }
    for (int b = 0; b < kTrLists; ++b) {
      mbar_init(smem_u32(&sm.list_full[b]), 1);
      mbar_init(smem_u32(&sm.list_free[b]), 19);         // all warps but 17
    }
    for (int t = 0; t < kTrTiles; ++t) {
      mbar_init(smem_u32(&sm.q_full[t]), 4);
      mbar_init(smem_u32(&sm.s_full[t]), 1);
      mbar_init(smem_u32(&sm.s_free[t]), 4);
      mbar_init(smem_u32(&sm.p_full[t]), 4);
      mbar_init(smem_u32(&sm.pv_done[t]), 1);
    }
    mbar_init(smem_u32(&sm.exch_full), 8);
    mbar_init(smem_u32(&sm.exch_free), 8);
    sm.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(&sm.tmem), kTrTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();
  bool bad = false;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  bool ok = true;

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTrRegsOther));
    if (warp == 17) {
      // ------------------------------------------------------- items and pages
      // units and items of all requests, summed
      long long all = 0, items = 0;
      int unit = 1;                                      // the longest slot
      TreeRequest r = {0, 0, 0, 0, 0};
      if (lane == 0) sm.upto[0] = sm.items[0] = 0;
#pragma unroll 1
      for (int i0 = 0; i0 < p.n; i0 += 32) {
        long long v = 0, w = 0;
        if (i0 + lane < p.n) {
          r = tree_request(p, i0 + lane, bad);
          const int slot = tr_slot(r, G);
          unit = max(unit, slot);
          w = static_cast<long long>(tr_groups(r, G) * p.Hkv) * slot;
          v = w * tr_steps(r);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long v0 = __shfl_up_sync(0xffffffffu, v, o), w0 = __shfl_up_sync(0xffffffffu, w, o);
          if (lane >= o) { v += v0; w += w0; }
        }
        if (i0 + lane < p.n) {
          sm.upto[i0 + lane + 1] = all + v;
          sm.items[i0 + lane + 1] = items + w;
        }
        all += __shfl_sync(0xffffffffu, v, 31);
        items += __shfl_sync(0xffffffffu, w, 31);
      }
      const int longest = __reduce_max_sync(0xffffffffu, unit);
      __syncwarp();
      const int before = static_cast<int>(min(static_cast<long long>(kTrSwitch), tr_divide(all + gridDim.x - 1, gridDim.x) / 2));       // slots of an item before its steps
      if (before) {
        for (int k = lane; k <= p.n; k += 32) sm.upto[k] += before * sm.items[k];
        all += before * items;
        __syncwarp();
      }
      const long long per = max(static_cast<long long>(longest), tr_divide(all + gridDim.x - 1, gridDim.x));
      long long u = min(all, per * blockIdx.x);
      const long long end = min(all, u + per);
      int i = 0, gs = 0;
      auto request_of = [&](int k) {                     // (the lanes have the first 32)
        if (p.n > 32) return tree_request(p, k, bad);
        TreeRequest to;
        to.slot = __shfl_sync(0xffffffffu, r.slot, k); to.row0 = __shfl_sync(0xffffffffu, r.row0, k); to.count = __shfl_sync(0xffffffffu, r.count, k);
        to.start = __shfl_sync(0xffffffffu, r.start, k); to.total = __shfl_sync(0xffffffffu, r.total, k);
        return to;
      };
      if (u < end) {                                     // the request of the first unit
        int hi = p.n;
        while (hi - i > 1) {
          const int mid = (i + hi) >> 1;
          if (sm.upto[mid] <= u) i = mid; else hi = mid;
        }
      }
      TrDesc d = {};
      int ids_next = 0;                                  // pages of the item made last, 32 from its first on
      auto ids_of = [&](const TrItem& l, int step) {
        const int at = (l.lo + step) * kTrPages + lane, pages = (l.total + kPageTokens - 1) / kPageTokens;
        return at < pages ? tree_page(p, l.slot, at, bad) : 0;
      };
      auto publish = [&](int n) {                        // the CTA's n-th item; false: there is none
        TrItem& to = sm.list[n % kTrLists];
        if (ok && n >= kTrLists) ok = tr_wait(smem_u32(&sm.list_free[n % kTrLists]), (n / kTrLists - 1) & 1, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return false;
        TrItem l;
        l.kvh = -1;
        while (u < end && l.kvh < 0) {
          while (u >= sm.upto[i + 1]) ++i;
          const TreeRequest of = request_of(i);
          const int S = tr_steps(of), groups = tr_groups(of, G), slot = tr_slot(of, G);
          const long long long_item = static_cast<long long>(slot) * (before + S), off = u - sm.upto[i];
          const int k = static_cast<int>(tr_divide(off, long_item));
          const long long item = u - (off - k * long_item);                              // where the item begins
          auto step_at = [&](long long at) {             // the first step whose slot begins at `at` or behind it
            return max(0, static_cast<int>(min((at - item + slot - 1) >> (slot - 1), static_cast<long long>(before + S))) - before);
          };
          const int s = step_at(u), n_steps = step_at(end) - s;
          u = min(end, item + long_item);
          if (n_steps <= 0) continue;
          l.kvh = k / groups;
          l.slot = of.slot; l.row0 = of.row0; l.count = of.count; l.start = of.start; l.total = of.total;
          l.first = (k - l.kvh * groups) * kTrItemRows;
          l.rows = min(kTrItemRows, of.count * G - l.first);
          l.lo = s;
          l.steps = of.total > 0 ? n_steps : 0;
          l.part = n_steps == S ? -1 : 2 * static_cast<int>(blockIdx.x) + (s == 0);
          if (l.part >= 0 && s == 0) {
            d.parts = static_cast<int>(tr_divide(item + slot * static_cast<long long>(before + S - 1), per)) - static_cast<int>(blockIdx.x) + 1;
            d.row0 = l.row0; d.first = l.first; d.rows = l.rows; d.kvh = l.kvh;
          }
          if (n > 0)                                     // its queries are on their way into the L2 cache
            for (int row = lane; row < l.rows; row += 32) {
              const int node = (l.first + row) / G;
              const __nv_bfloat16* at = p.q + (l.row0 + node) * p.ldq + (l.kvh * G + (l.first + row - node * G)) * kD;
              asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
              asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 64));
            }
        }
        if (lane == 0) {
          to = l;
          sm.redo[n % kTrLists] = 0;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.list_full[n % kTrLists]));
        if (l.kvh >= 0) ids_next = ids_of(l, 0);
        return l.kvh >= 0;
      };
      TrItem l = {};
      int pages = 0, ids = 0, ids_later = 0;
#pragma unroll 1
      for (int it = -1;; ++it) {                         // (-1: nothing yet but the first item)
        bool more = false;
        int s = 0;
#pragma unroll 1
        do {
          if (s < l.steps) {
            if (s > 0 && s % 8 == 0) ids = ids_later;
            const int b = gs % kTrRaw;
            if (ok && gs >= kTrRaw) ok = tr_wait(smem_u32(&sm.raw_free[b]), (gs / kTrRaw - 1) & 1, abort_flag, limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int n = min(kTrPages, pages - (l.lo + s) * kTrPages);
            if (lane == 0) mbar_expect_tx(smem_u32(&sm.raw_full[b]), n * L::bytes);
            __syncwarp();
            const int page = __shfl_sync(0xffffffffu, ids, (s % 8) * kTrPages + (lane & 3));
            if (lane < n)
              bulk_g2s(smem_u32(raw + (b * kTrPages + lane) * L::stride), p.cache + (static_cast<size_t>(page) * p.Hkv + l.kvh) * L::bytes, L::bytes, smem_u32(&sm.raw_full[b]));
            if (s % 8 == 0 && s + 8 < l.steps) ids_later = ids_of(l, s + 8);
            ++gs;
          }
          if (s == max(0, min(1, l.steps - 1))) more = publish(it + 1);
        } while (++s < l.steps);
        if (!more || !ok) break;
        l = sm.list[(it + 1) % kTrLists];
        pages = (l.total + kPageTokens - 1) / kPageTokens;
        ids = ids_next;
      }
      if (lane == 0) desc[blockIdx.x] = d;
      if (*abort_flag) {                                 // copies in flight land (for a bounded time) before the CTA goes
        const long long t0 = clock64();
        for (int g = max(0, gs - kTrRaw); g < gs; ++g)
          while (!mbar_try_wait(smem_u32(&sm.raw_full[g % kTrRaw]), (g / kTrRaw) & 1) && clock64() - t0 < kWaitBudgetCycles / 8) {
          }
      }
    } else if (warp == 19) {
      // ------------------------------------------------------ powers of two
      TrRing raw_at(kTrRaw), note_at(kTrNotes);
#pragma unroll 1
      for (int it = 0;; ++it) {
        const TrItem& l = sm.list[it % kTrLists];
        if (ok) ok = tr_wait(smem_u32(&sm.list_full[it % kTrLists]), (it / kTrLists) & 1, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok || l.kvh < 0) break;
        const int steps = l.steps;
        int v_exp = 0, visible = l.total - l.lo * kTrTok, v_most = -200, v_least = 200;              // of the item's steps
        bool v_wide = false;
#pragma unroll 1
        for (int s = 0; s < steps; ++s, visible -= kTrTok) {
          if (ok) ok = tr_wait(smem_u32(&sm.raw_full[raw_at.i]), raw_at.phase, abort_flag, limit);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint8_t* pages = raw + raw_at.i * kTrPages * L::stride;
          uint32_t most[2] = {0u, 0u}, least[2] = {0u, 0u};
          bool odd = false;                              // some are not finite
          const uint8_t* of = pages + L::vScale;
#pragma unroll 1
          for (int w = 1; w >= 0; --w) {                 // V, then K
            float4 scale[2];
            pf_scales(of, L::stride, visible, lane, scale);
            of = pages + L::kScale;
            most[1] = most[0];
            least[1] = least[0];
            most[0] = __reduce_max_sync(0xffffffffu, max(pf_most<false>(scale[0]), pf_most<false>(scale[1])));
            if (__builtin_expect(most[0] >= 0x7F800000u, 0)) {
              odd = true;
              most[0] = __reduce_max_sync(0xffffffffu, max(pf_most<true>(scale[0]), pf_most<true>(scale[1])));
            }
            least[0] = __reduce_min_sync(0xffffffffu, min(tr_least(scale[0]), tr_least(scale[1])));
          }
          const int ek = pf_exponent(most[0]), ev = pf_exponent(most[1]), lk = pf_exponent(least[0]);
          const bool k_wide = lk < ek - kTrApart || ek > 100;
          v_most = max(v_most, ev);
          v_least = min(v_least, pf_exponent(least[1]));
          // V: one unit for the item, that follows the largest scale; in the long conversion only when operands pass 2^15
          if (!v_wide) {
            v_exp = v_most + 10;
            if (v_least < v_most - kTrApart || v_most > 100) { v_wide = true; v_exp = v_most - 3; }
          } else if (ev - 7 > v_exp) {
            v_exp = ev - 3;
          }
          if (lane == 0) {
            if (odd || lk < ek - kTrApartK || v_least < v_most - kTrApartV) sm.redo[it % kTrLists] = 1;
            auto& to = sm.note[note_at.i];
            to.k = pow2f(k_wide ? 5 - ek : 14 - ek);
            to.v = pow2f(v_wide ? -v_exp : 24 - v_exp);
            to.k_wide = k_wide;
            to.v_wide = v_wide;
            to.back = pow2f(k_wide ? ek - 5 : ek + 10);
            to.v_exp = v_exp;
            mbar_arrive(smem_u32(&sm.note_full[note_at.i]));
          }
          __syncwarp();
          raw_at.advance();
          note_at.advance();
        }
        if (lane == 0) mbar_arrive(smem_u32(&sm.list_free[it % kTrLists]));
      }
    } else {
      // ---------------------------------------------------------------- MMAs
      const bool leader = elect_one();
      const int t = warp == 18;
      const uint32_t idesc_s = umma_idesc(kTrRows, kTrTok, 0u, 0u), idesc_o = umma_idesc(kTrRows, kD, 0u, 0u) | 1u << 16;      // V: channels are contiguous
      const uint64_t dq = umma_desc_sw128(smem_u32(sm.q[t])), dk = umma_desc_sw128(smem_u32(sm.k[0])), dv = umma_desc_sw128_n(smem_u32(sm.v[0]), kTrHalf);
      const uint32_t tile = tmem + t * kTrTmemTile;
      int before = 0;                                    // steps of earlier items
      uint32_t q_phase = 0, k_phase = 0, v_phase = 0, s_phase = 1, p_phase = 0;            // k and v: bit = place; (a wait for scores that nobody holds is over at once)
#pragma unroll 1
      for (int it = 0;; ++it) {
        const TrItem& l = sm.list[it % kTrLists];
        if (ok) ok = tr_wait(smem_u32(&sm.list_full[it % kTrLists]), (it / kTrLists) & 1, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok || l.kvh < 0) break;
        const int steps = l.steps, first = tr_first(l, t, before);
        const bool split = tr_split(l);
        const int by = split ? 2 : 1;
        if (first < steps) {
          if (ok) ok = tr_wait(smem_u32(&sm.q_full[t]), q_phase, abort_flag, limit);
          q_phase ^= 1u;
        }
        // scores of step s, then the product of the one before: scores run ahead of their softmax
#pragma unroll 1
        for (int s = first; s < steps + by && first < steps; s += by) {
          if (s < steps) {
            const int b = (before + s) & (kTrOpsK - 1);
            if (ok) ok = tr_wait(smem_u32(&sm.k_full[t][b]), k_phase >> b & 1, abort_flag, limit);
            if (ok) ok = tr_wait(smem_u32(&sm.s_free[t]), s_phase, abort_flag, limit);
            ok = __all_sync(0xffffffffu, ok);
            k_phase ^= 1u << b;
            s_phase ^= 1u;
            tc_fence_after();
            if (ok && leader) {
              const uint64_t k0 = dk + (b * (2 * kTrHalf) >> 4);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16_ts(tile, tile + kTrTmemQ + k * 8, k0 + k * 2, idesc_s, k > 0);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16(tile, dq + k * 2, k0 + (kTrHalf >> 4) + k * 2, idesc_s, 1);
              tc_commit(smem_u32(&sm.s_full[t]));
              tc_commit(smem_u32(&sm.k_free[b]));
              if (split) tc_commit(smem_u32(&sm.k_free[b]));
            }
            __syncwarp();
          }
          if (s > first) {
            const int b = (before + s - by) & (kTrOpsV - 1);
            if (ok) ok = tr_wait(smem_u32(&sm.v_full[t][b]), v_phase >> b & 1, abort_flag, limit);
            if (ok) ok = tr_wait(smem_u32(&sm.p_full[t]), p_phase, abort_flag, limit);
            ok = __all_sync(0xffffffffu, ok);
            v_phase ^= 1u << b;
            p_phase ^= 1u;
            tc_fence_after();
            if (ok && leader) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ts(tile + kTrTmemO, tile + kTrTmemP + k * 8, dv + (b * (2 * kTrHalf) >> 4) + k * (16 * 128 >> 4), idesc_o, s - by > first || k > 0);
              tc_commit(smem_u32(&sm.pv_done[t]));
              tc_commit(smem_u32(&sm.v_free[b]));
              if (split) tc_commit(smem_u32(&sm.v_free[b]));
            }
            __syncwarp();
          }
        }
        before += steps;
        if (lane == 0) mbar_arrive(smem_u32(&sm.list_free[it % kTrLists]));
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ conversion
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTrRegsConvert));
    // warps 8-11 take the even steps, 12-15 the odd ones, K first: scores run ahead of their softmax
    const int ct = tid & 127, mine = warp >= 12;
    TrRing raw_at(kTrRaw, 0, mine), note_at(kTrNotes, 0, mine);
    uint32_t k_phase = 1, v_phase = 1;                   // (a wait for operands that nobody reads is over at once)
    int vb = mine;                                       // V's place
    int ahead = mine;                                    // steps from the item's first to this warp's next
#pragma unroll 1
    for (int it = 0;; ++it) {
      const TrItem& l = sm.list[it % kTrLists];
      if (ok) ok = tr_wait(smem_u32(&sm.list_full[it % kTrLists]), (it / kTrLists) & 1, abort_flag, limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok || l.kvh < 0) break;
      const int steps = l.steps;
      const bool split = tr_split(l);
      int visible = l.total - (l.lo + ahead) * kTrTok;
#pragma unroll 1
      for (; ahead < steps; ahead += 2, visible -= 2 * kTrTok) {
        if (ok) ok = tr_wait(smem_u32(&sm.raw_full[raw_at.i]), raw_at.phase, abort_flag, limit);
        if (ok) ok = tr_wait(smem_u32(&sm.note_full[note_at.i]), note_at.phase, abort_flag, limit);
        if (ok) ok = tr_wait(smem_u32(&sm.k_free[mine]), k_phase, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* pages = raw + raw_at.i * kTrPages * L::stride;
        const auto& note = sm.note[note_at.i];
        const float v_mul = note.v;
        const int v_wide = note.v_wide;
        if (__builtin_expect(!note.k_wide, 1)) tr_convert_k<KBITS, VBITS, false>(sm.k[mine], pages, note.k, ct);
        else tr_convert_k<KBITS, VBITS, true>(sm.k[mine], pages, note.k, ct);
        fence_proxy_async_smem();
        __syncwarp();
        // (of items in both tiles, the even steps are tile 0's)
        if (lane == 0) {
          mbar_arrive(smem_u32(&sm.k_full[mine][mine]));
          if (!split) mbar_arrive(smem_u32(&sm.k_full[1 - mine][mine]));
        }
        ok = tr_wait(smem_u32(&sm.v_free[vb]), v_phase, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (__builtin_expect(!v_wide, 1)) tr_convert_v<KBITS, VBITS, false>(sm.v[vb], pages, visible, v_mul, ct);
        else tr_convert_v<KBITS, VBITS, true>(sm.v[vb], pages, visible, v_mul, ct);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sm.v_full[mine][vb]));
          if (!split) mbar_arrive(smem_u32(&sm.v_full[1 - mine][vb]));
          mbar_arrive(smem_u32(&sm.raw_free[raw_at.i]));
        }
        raw_at.advance(2);
        note_at.advance(2);
        k_phase ^= 1u;
        vb ^= 2;
        v_phase ^= vb == mine;
      }
      ahead -= steps;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.list_free[it % kTrLists]));
    }
  } else {
    // --------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTrRegsSoftmax));
    const int t = warp >> 2, row = tid & 127;
    const uint32_t tile = tmem + t * kTrTmemTile + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    struct Row {
      long long q, out;                                  // where its query and result are; q < 0: not a row
      const uint32_t* sees;
      float mul;                                         // what its scores are multiplied with, but for K's power of two
    };
    // the row of the thread in item `it`, and Q of its tile; false: no more items
    auto begin = [&](int it, int before, Row& r) {
      const TrItem& l = sm.list[it % kTrLists];
      if (ok) ok = tr_wait(smem_u32(&sm.list_full[it % kTrLists]), (it / kTrLists) & 1, abort_flag, limit);
      ok = __all_sync(0xffffffffu, ok);
      r.q = r.out = -1;
      r.sees = p.masks;
      r.mul = 0.f;
      if (!ok || l.kvh < 0) return false;
      const int at = tr_split(l) ? row : t * kTrRows + row;
      if (at < l.rows) {
        const int node = (l.first + at) / G, col = (l.kvh * G + (l.first + at - node * G)) * kD;
        r.q = (l.row0 + node) * p.ldq + col;
        r.out = (l.row0 + node) * p.ldo + col;
        r.sees = p.masks + (l.row0 + node) * p.ldm;
      }
      if (tr_first(l, t, before) < l.steps) {
        // a power of two brings the row's largest magnitude to 2^10 .. 2^11; what is not finite stays
        // All loads in flight at once, eight lanes a row (a row a lane would have 32 lines of memory in a load: 7000 cycles, not 2500); a half at a time goes to the
        // row's lane by way of the warp's own rows of Q's operand.
        uint4 q[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const long long from = __shfl_sync(0xffffffffu, r.q, 4 * j + (lane >> 3));
#pragma unroll
          for (int h = 0; h < 2; ++h) q[8 * h + j] = from >= 0 ? reinterpret_cast<const uint4*>(p.q + from)[8 * h + (lane & 7)] : make_uint4(0u, 0u, 0u, 0u);
        }
        uint8_t* rows = sm.q[t] + (warp & 3) * 32 * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int of = 4 * j + (lane >> 3);
            *reinterpret_cast<uint4*>(rows + of * 128 + (((lane & 7) ^ (of & 7)) << 4)) = q[8 * h + j];
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 8; ++c) q[8 * h + c] = *reinterpret_cast<const uint4*>(rows + lane * 128 + ((c ^ (lane & 7)) << 4));
          __syncwarp();
        }
        uint32_t most = 0;                               // (two magnitudes a word: the larger of the upper, then of the lower ones)
#pragma unroll
        for (int c = 0; c < 16; ++c) most = __vmaxu2(most, __vmaxu2(__vmaxu2(q[c].x & 0x7FFF7FFFu, q[c].y & 0x7FFF7FFFu), __vmaxu2(q[c].z & 0x7FFF7FFFu, q[c].w & 0x7FFF7FFFu)));
        most = max(most >> 16, most & 0xFFFFu);
        const int e = most >= 0x7F80u || most == 0u ? 0 : max(static_cast<int>(most >> 7) - 127 - 10, -126);
        const float down = pow2f(-e);
        r.mul = pow2f(e) * p.scale * 1.4426950408889634f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {                   // eight channels
          const uint32_t in[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&in[j]));
            x[j] = pack_f16x2(f.x * down, f.y * down);
          }
          if (c < 8) tr_tmem_st4(tile + kTrTmemQ + c * 4, x);
          else *reinterpret_cast<uint4*>(sm.q[t] + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
        }
        tmem_st_wait();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full[t]));
      }
      return true;
    };
    int before = 0, n = 0, exchanges = 0;                // steps of earlier items; steps that this tile took part in; items in both tiles
    bool lent = false;                                   // the other tile may still read this one's output
    auto wait_lent = [&]() {
      if (lent && ok) ok = tr_wait(smem_u32(&sm.exch_free), (exchanges - 1) & 1, abort_flag, limit);
      lent = false;
    };
    Row cur = {-1, -1, p.masks, 0.f};
    bool more = true;
#pragma unroll 1
    for (int it = -1; more; ++it) {                      // (-1: nothing yet but the first item's Q)
      const TrItem& l = sm.list[max(it, 0) % kTrLists];
      const int steps = it < 0 ? 0 : l.steps, start = l.start, total = l.total;
      const int first = it < 0 ? 0 : tr_first(l, t, before);
      const bool split = it >= 0 && tr_split(l), in = first < steps, mine = cur.q >= 0;
      float m = -INFINITY, sum = 0.f;
      int v_exp = 0;
      {
#pragma unroll 1
        for (int s = first; s < steps; s += split ? 2 : 1) {
          const int tok0 = (l.lo + s) * kTrTok, note = (before + s) & (kTrNotes - 1);
          if (ok) ok = tr_wait(smem_u32(&sm.s_full[t]), n & 1, abort_flag, limit);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          if (__builtin_expect(tok0 + kTrTok > start, 0)) {                   // what a row does not see: -inf in place of its scores
            const uint2 see = mine ? tr_visible(cur.sees, p.words, start, total, tok0) : make_uint2(0u, 0u);
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t a[32];
              tmem_ld_32x32(tile + c * 32, a);
              tmem_ld_wait();
              const uint32_t bits = c == 0 ? see.x : see.y;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(bits >> j & 1u)) a[j] = 0xFF800000u;
              tmem_st_32x32(tile + c * 32, a);
            }
            tmem_st_wait();
          }
          // all scores into registers: the next step's replace them at once (2 x 64 behind 32000: 101 us; with the scores read again for the exponentials 109)
          uint32_t a[2][32];
          tmem_ld_32x32(tile, a[0]);
          tmem_ld_32x32(tile + 32, a[1]);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.s_free[t]));
          float of[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 64; j += 2) of[j / 2 & 3] = fmaxf(of[j / 2 & 3], fmaxf(__uint_as_float(a[j >> 5][j & 31]), __uint_as_float(a[j >> 5][(j & 31) + 1])));
          const float mx = fmaxf(fmaxf(of[0], of[1]), fmaxf(of[2], of[3]));
          // (there before K was converted; written again after this step's product, which waits for what follows: kTrNotes)
          const float2 told = make_float2(sm.note[note].back, __int_as_float(sm.note[note].v_exp));
          const float mul = told.x * cur.mul, top = mx * mul;
          float alpha = 1.f;
          bool grew = top > m + kTrGrowth || (m == -INFINITY && top > m);
          if (grew) {
            alpha = fast_exp2(m - top);
            m = top;
            sum *= alpha;
          }
          const int e = __float_as_int(told.y);
          if (e != v_exp) {
            alpha = v_exp - e < -126 ? 0.f : alpha * pow2f(v_exp - e);
            v_exp = e;
            grew = true;
          }
          const float use = m == -INFINITY ? 0.f : m;
          const float2 less = make_float2(-use, -use), mul2 = make_float2(mul, mul);
          // the previous product has read the probabilities and written the output
          if (ok && s > first) ok = tr_wait(smem_u32(&sm.pv_done[t]), (n - 1) & 1, abort_flag, limit);
          if (s == first) wait_lent();
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          float2 part_sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pr[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {                // (f16: off by 2^-11 of itself, below 2^-14 by 2^-25; their sum has them as they are)
              const int at = c * 16 + 2 * j;
              const float2 d = __ffma2_rn(make_float2(__uint_as_float(a[at >> 5][at & 31]), __uint_as_float(a[at >> 5][(at & 31) + 1])), mul2, less);
              const float2 x = make_float2(fast_exp2(d.x), fast_exp2(d.y));
              part_sum[j & 1] = __fadd2_rn(part_sum[j & 1], x);
              pr[j] = pack_f16x2(x.x, x.y);
            }
            tr_tmem_st8(tile + kTrTmemP + c * 8, pr);
          }
          sum += (part_sum[0].x + part_sum[0].y) + (part_sum[1].x + part_sum[1].y);
          if (__builtin_expect(s > first && __any_sync(0xffffffffu, grew), 0)) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld_32x32(tile + kTrTmemO + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st_32x32(tile + kTrTmemO + c * 32, o);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[t]));
          ++n;
        }
      }
      // the next item's Q while the last product runs (all of this item's scores are there)
      Row next;
      more = begin(it + 1, before + steps, next);
      const int part = it < 0 ? -1 : l.part;
      // of a part, [four channels][row]: a warp's rows are neighbours
      const size_t in_part = split ? row : t * kTrRows + row, at = static_cast<size_t>(max(part, 0)) * part_rows + in_part;
      float4* const part_to = reinterpret_cast<float4*>(part_o) + static_cast<size_t>(max(part, 0)) * 32 * part_rows + in_part;
      if (steps == 0) {                                  // a request that is told wrongly
        if (mine) {
#pragma unroll
          for (int j = 0; j < 16; ++j) reinterpret_cast<uint4*>(p.out + cur.out)[j] = make_uint4(0u, 0u, 0u, 0u);
        }
      } else {
        if (ok && in) ok = tr_wait(smem_u32(&sm.pv_done[t]), (n - 1) & 1, abort_flag, limit);
        ok = __all_sync(0xffffffffu, ok);
        // what this tile's output and the other's are multiplied with
        float mul[2] = {pow2f(v_exp), 0.f};
        const bool other = split && (1 - first) < steps; // the other tile has an output
        if (split) {
          wait_lent();
          sm.exch_ml[t][row] = make_float2(m, sum);
          sm.exch_exp[t][row] = v_exp;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.exch_full));
          if (ok) ok = tr_wait(smem_u32(&sm.exch_full), exchanges & 1, abort_flag, limit);
          ok = __all_sync(0xffffffffu, ok);
          ++exchanges;
          lent = true;
          const float2 o = sm.exch_ml[1 - t][row];
          const float top = fmaxf(m, o.x), use = top == -INFINITY ? 0.f : top, f0 = fast_exp2(m - use), f1 = fast_exp2(o.x - use);
          mul[0] *= f0;
          mul[1] = f1 * pow2f(sm.exch_exp[1 - t][row]);
          sum = f0 * sum + f1 * o.y;
          m = top;
        }
        tc_fence_after();
        if (!*const_cast<volatile uint32_t*>(&sm.redo[it % kTrLists])) {
          const float inv = part >= 0 ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;            // NaN stays
          const long long beside = __shfl_xor_sync(0xffffffffu, cur.out, 1);                              // the next lane's row
          const int c0 = split ? 4 * t : 0, c1 = split ? 4 * t + 4 : 8;                                  // of 16 channels
#pragma unroll 1
          for (int c = c0; c < c1; ++c) {
            uint32_t a[16], b[16];
            const uint32_t from = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + kTrTmemO + c * 16;
            if (in) tmem_ld_32x16(from + t * kTrTmemTile, a);
            if (other) tmem_ld_32x16(from + (1 - t) * kTrTmemTile, b);
            tmem_ld_wait();
            float o[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              o[j] = in ? __uint_as_float(a[j]) * mul[0] : 0.f;
              if (other) o[j] = fmaf(__uint_as_float(b[j]), mul[1], o[j]);
              o[j] *= inv;
            }
            if (mine && part >= 0) {
#pragma unroll
              for (int j = 0; j < 4; ++j) part_to[static_cast<size_t>(4 * c + j) * part_rows] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            } else if (part < 0) {
              // two lanes write a row's 32 bytes, then the next row's
              const uint4 x = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])),
                          y = make_uint4(pack_bf16x2(o[8], o[9]), pack_bf16x2(o[10], o[11]), pack_bf16x2(o[12], o[13]), pack_bf16x2(o[14], o[15]));
              const bool odd = lane & 1;
              uint4 z = odd ? x : y;
              z.x = __shfl_xor_sync(0xffffffffu, z.x, 1); z.y = __shfl_xor_sync(0xffffffffu, z.y, 1);
              z.z = __shfl_xor_sync(0xffffffffu, z.z, 1); z.w = __shfl_xor_sync(0xffffffffu, z.w, 1);
              const long long even_row = odd ? beside : cur.out, odd_row = odd ? cur.out : beside;
              if (even_row >= 0) *reinterpret_cast<uint4*>(p.out + even_row + c * 16 + 8 * odd) = odd ? z : x;
              if (odd_row >= 0) *reinterpret_cast<uint4*>(p.out + odd_row + c * 16 + 8 * odd) = odd ? y : z;
            }
          }
          if (part >= 0 && mine && c0 == 0) part_ml[at] = make_float2(m, sum);
        } else if (ok) {
          TreeRequest r;
          r.slot = l.slot; r.row0 = l.row0; r.count = l.count; r.start = start; r.total = total;
          const int lo = l.lo * kTrTok, hi = min(total, (l.lo + steps) * kTrTok);
#pragma unroll 1
          for (uint32_t rows = __ballot_sync(0xffffffffu, mine && (!split || (lane & 1) == t)); rows; rows &= rows - 1) {
            const int of = __ffs(rows) - 1;
            const long long q = __shfl_sync(0xffffffffu, cur.q, of), out = __shfl_sync(0xffffffffu, cur.out, of);
            const uint32_t* sees = reinterpret_cast<const uint32_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(cur.sees), of));
            float rm, rs, o[4];
            tree_row<KBITS, VBITS>(p, r, l.kvh, lo, hi, sees, p.q + q, lane, rm, rs, o, bad);
            if (part >= 0) {
              part_to[static_cast<size_t>(lane) * part_rows - lane + of] = make_float4(o[0], o[1], o[2], o[3]);
              if (lane == 0) part_ml[at - lane + of] = make_float2(rm, rs);
            } else {
              const float f = rs > 0.f ? 1.f / rs : rs == 0.f ? 0.f : rs;
              reinterpret_cast<uint2*>(p.out + out)[lane] = make_uint2(pack_bf16x2(o[0] * f, o[1] * f), pack_bf16x2(o[2] * f, o[3] * f));
            }
          }
        }
        tc_fence_before();
        if (split) {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.exch_free));
        }
      }
      __syncwarp();
      if (lane == 0 && it >= 0) mbar_arrive(smem_u32(&sm.list_free[it % kTrLists]));
      before += steps;
      cur = next;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) tmem_dealloc(tmem, kTrTmemCols);
  if (bad) atomicExch(p.status, static_cast<uint32_t>(kErrBadArgument));
  if (tid == 0 && sm.abort_word) atomicExch(p.status, static_cast<uint32_t>(kErrBarrierTimeout));
}

// Joins the parts of items that several CTAs shared: block x looks after the item that began in CTA x and went on beyond it.  A warp's lanes are eight rows times four of
// the 32 fours of channels, so that both sides are whole sectors; a thread has ROWS rows, eight apart, and PARTS parts of them in flight.  Few rows mean many parts of each
// and blocks that are all resident at once: one row and eight parts (1 x 8 behind 700: 15.4 us, with two and four 17.8); else two and four (2 x 64 behind 32000: 109.6 us
// against 110.9, 32 x 64 behind up to 1500: 122.6 against 126.3).
static constexpr int kTrMergeFew = 40;                   // rows: five blocks fit a multiprocessor
template <int ROWS, int PARTS>
__global__ void __launch_bounds__(256)
tree_merge_kernel(const CbTreeAttn p, const int part_rows) {
  pdl_wait();
  pdl_launch_dependents();
  const float4* part_o = reinterpret_cast<const float4*>(p.partial);
  const float2* part_ml = reinterpret_cast<const float2*>(part_o + static_cast<size_t>(gridDim.x) * 2 * part_rows * (kD / 4));
  const TrDesc d = reinterpret_cast<const TrDesc*>(part_ml + static_cast<size_t>(gridDim.x) * 2 * part_rows)[blockIdx.x];
  const int row0 = blockIdx.y * 8 * ROWS + (threadIdx.x & 7), four = threadIdx.x >> 3, G = p.Hq / p.Hkv;
  if (d.parts <= 0 || row0 >= d.rows) return;
  float m[ROWS], sum[ROWS], o[ROWS][4];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    m[k] = -INFINITY;
    sum[k] = o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
  }
#pragma unroll 1
  for (int c = 0; c < d.parts; c += PARTS) {
    float2 ml[PARTS][ROWS];
    float4 x[PARTS][ROWS];
#pragma unroll
    for (int e = 0; e < PARTS; ++e) {
      const size_t part = 2 * (blockIdx.x + c + e) + (c + e == 0);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int row = row0 + 8 * k;
        const bool there = c + e < d.parts && row < d.rows;
        ml[e][k] = there ? __ldcg(part_ml + part * part_rows + row) : make_float2(-INFINITY, 0.f);
        x[e][k] = there ? __ldcg(part_o + (part * 32 + four) * part_rows + row) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      float top = m[k];
#pragma unroll
      for (int e = 0; e < PARTS; ++e) top = fmaxf(top, ml[e][k].x);
      const float use = top == -INFINITY ? 0.f : top, old = fast_exp2(m[k] - use);
      m[k] = top;
      sum[k] *= old;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[k][j] *= old;
#pragma unroll
      for (int e = 0; e < PARTS; ++e) {
        const float f = fast_exp2(ml[e][k].x - use);     // of a part that saw nothing: zero
        sum[k] = fmaf(f, ml[e][k].y, sum[k]);
        o[k][0] = fmaf(f, x[e][k].x, o[k][0]);
        o[k][1] = fmaf(f, x[e][k].y, o[k][1]);
        o[k][2] = fmaf(f, x[e][k].z, o[k][2]);
        o[k][3] = fmaf(f, x[e][k].w, o[k][3]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int row = row0 + 8 * k;
    if (row >= d.rows) break;
    const float f = sum[k] > 0.f ? 1.f / sum[k] : sum[k] == 0.f ? 0.f : sum[k];
    const int node = (d.first + row) / G;
    const long long to = (d.row0 + node) * p.ldo + (d.kvh * G + (d.first + row - node * G)) * kD + four * 4;
    *reinterpret_cast<uint2*>(p.out + to) = make_uint2(pack_bf16x2(o[k][0] * f, o[k][1] * f), pack_bf16x2(o[k][2] * f, o[k][3] * f));
  }
}

template <int KB, int VB>
static int launch_tree(const CbTreeAttn& p, cudaStream_t st) {
  const size_t smem = sizeof(TrSmem) + 1024 + static_cast<size_t>(kTrRaw) * kTrPages * TreeLay<KB, VB>::stride;
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -18;
  if (!sms[dev]) {
    cudaError_t e = cudaFuncSetAttribute(tree_kernel<KB, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    int n = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<int>(e);
    // the warps' new shares come out of the registers that the block was launched with
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, tree_kernel<KB, VB>);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (at.numRegs < kTrRegs) return -19;
    sms[dev] = n;
  }
  const int rows = tr_rows(p.words, p.rows, p.Hq / p.Hkv);
  cudaError_t e = launch(tree_kernel<KB, VB>, dim3(sms[dev]), dim3(kTrThreads), smem, st, p, rows, tr_limit(p));
  const int step = rows <= kTrMergeFew ? 8 : 16;
  if (e == cudaSuccess) e = launch(step == 8 ? tree_merge_kernel<1, 8> : tree_merge_kernel<2, 4>, dim3(sms[dev], (rows + step - 1) / step), dim3(256), 0, st, p, rows);
  return static_cast<int>(e);
}

}  // namespace cb

extern "C" {

// fp32 scratch elements of a launch on a GPU of `sms` multiprocessors
long long cb_tree_attn_floats(int sms, int words, int rows, int group) {
  return static_cast<long long>(sms) * (2 * cb::tr_rows(words, rows, group) * (cb::kD + 2) + static_cast<long long>(sizeof(cb::TrDesc) / 4));
}

int cb_tree_attn(const CbTreeAttn* p, void* stream) {
  using namespace cb;
  if (p->n <= 0 || p->rows <= 0) return 0;
  if (p->n > kTreeMaxRequests || p->words < 1 || p->words > kTreeMaxWords || p->Hkv <= 0 || p->Hq % p->Hkv != 0 || p->Hq / p->Hkv > kTreeMaxGroup || p->width > 1 << 26) return -10;
  if (!p->partial) return -12;
  return with_kv_bits(p->k_bits, p->v_bits, [&](auto kb, auto vb) { return launch_tree<decltype(kb)::value, decltype(vb)::value>(*p, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
