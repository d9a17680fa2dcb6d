// Logits as the requests want them: penalties for repeated tokens, biases of chosen tokens, masks of grammars.
//
// For token t of a row: s = whether the request's prompt or output holds it, c = how often its output does (with the drafts that lead to the row), b its bias:
//   x = logit;  s: x = x > 0 ? x / repetition : x * repetition;  x -= frequency * c;  c > 0: x -= presence;  x += b;  not allowed: x = -inf
// in fp32, rounded once to the type of the logits.
//
// Bound by memory: a row is read and written once, 16 bytes at a time.  A block has a range of a row's tokens (16 KB of logits).  With its logits on their way it reads
// the request's history, which is in the caches for the row's other blocks, and marks the tokens of its range that are in it; the first to mark one clears its word.
// Then the logits are copied (in place: left), the words count, and the marked tokens are done by a thread each: few of a range are, but most warps would meet one (all
// tokens through their words: 223 us for 624 rows of 151936, so 104, 3.6 TB/s).  256 rows of 151936 behind 1280 tokens, with biases and some masks, from one buffer to
// another: 53 us, 2.9 TB/s; in place without masks, where only the marked tokens are touched, 30; 624 rows of trees in place 71; one row 5.
#include "ptx.cuh"
#include "launch.cuh"

// Packed by ops/native.py::ADJUST.
struct CbAdjust {
  const void* logits;        // [rows, vocab] bf16 or fp32, row stride ldl
  void* out;                 // likewise, ldo; may be `logits`
  const int* request;        // [rows] request of a row, below 0: none
  const int* history;        // [n, most], row stride ldh
  const int* length;         // [n] tokens of the history
  const int* prompt;         // [n] how many of them are the prompt's
  const float* repetition;   // [n] or null
  const float* frequency;
  const float* presence;
  const int* bias_at;        // [n + 1] or null: the request's entries of
  const int* bias_id;        // [biases]
  const float* bias;
  const uint32_t* mask;      // [rows] words of 32 tokens, row stride ldm, or null
  const int* draft;          // [rows] tokens of the nodes, or null
  const uint32_t* sees;      // [rows, words], row stride lds: the nodes above a node, and itself
  const int* row0;           // [n] row of the request's node 0, whose token is in the history
  long long ldl, ldo, ldh, ldm, lds;
  int rows, vocab, n, most, biases, words, f32;
};

namespace cb {

// A token's word: index of its bias + 1 (kAdjustFar: at least that), seen, count
static constexpr uint32_t kAdjustFar = 2047u, kAdjustSeen = 1u << 11, kAdjustOne = 1u << 12;
static constexpr int kAdjustBytes = 16384;               // of a block's logits

static_assert(kAdjustBytes / 2 / 32 <= 256, "a word of marks for every thread");
static constexpr int kAdjustList = 1024, kAdjustAhead = 2;

__device__ __forceinline__ float adjust_load(float v) { return v; }
__device__ __forceinline__ float adjust_load(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void adjust_store(float& to, float v) { to = v; }
__device__ __forceinline__ void adjust_store(__nv_bfloat16& to, float v) { to = __float2bfloat16(v); }

// THREADS: 256, so that six blocks of an SM have their latencies at different times, or 1024 where there are no more than two blocks an SM: then the trips through a
// long history count (9 rows of 50257 behind 20000 tokens: 29 us by blocks of 256).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS)
adjust_kernel(const CbAdjust p) {
  constexpr int N = 16 / sizeof(T), kRange = kAdjustBytes / sizeof(T), kVectors = kAdjustBytes / 16 / THREADS;
  __shared__ uint32_t table[kRange], marked[kRange / 32];
  __shared__ uint16_t list[kAdjustList];
  __shared__ int listed;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* in = static_cast<const T*>(p.logits) + row * p.ldl;
  T* out = static_cast<T*>(p.out) + row * p.ldo;
  // ranges start where the logits do on 16 bytes: the first begins up to N - 1 tokens before the row
  const int ahead = static_cast<int>(reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T), lo = blockIdx.x * kRange - ahead;
  if (lo >= p.vocab) return;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == (reinterpret_cast<uintptr_t>(in) & 15), copies = in != out || p.mask != nullptr;
  uint4 v[kVectors];
  if (copies) {
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      const int at = lo + (k * THREADS + tid) * N;
      if (at >= 0 && at + N <= p.vocab) v[k] = *reinterpret_cast<const uint4*>(in + at);
    }
  }
  const int r = p.request != nullptr ? p.request[row] : row;
  const bool known = r >= 0 && r < p.n;
  int length = 0, prompt = 0, b0 = 0, b1 = 0, row0 = -1;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (known) {
    length = min(max(p.length[r], 0), p.most);
    if (p.prompt != nullptr) prompt = p.prompt[r];
    if (p.bias_at != nullptr) { b0 = max(p.bias_at[r], 0); b1 = min(p.bias_at[r + 1], p.biases); }
    if (p.draft != nullptr) row0 = p.row0[r];
    if (p.repetition != nullptr) rep = p.repetition[r];
    if (p.frequency != nullptr) freq = p.frequency[r];
    if (p.presence != nullptr) pres = p.presence[r];
  }
  for (int i = tid; i < kRange / 32; i += THREADS) marked[i] = 0;
  if (tid == 0) listed = 0;
  __syncthreads();
  const int* said = known ? p.history + r * p.ldh : p.history;
  const int first = min(length, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(said) & 15)) & 15) / 4);       // up to the first 16 bytes
  const int fours = (length - first) / 4;
  const int from = max(lo, 0);                             // the range's tokens that there are
  const unsigned tokens = min(lo + kRange, p.vocab) - from;
  // f(place in the range, whether it is the output's) for the tokens of the history and the drafts above the row; in this block's range
  auto each = [&](auto f) {
    auto one = [&](int token, bool own) {
      if (static_cast<unsigned>(token - from) < tokens) f(token - lo, own);
    };
    if (tid < first) one(said[tid], tid >= prompt);
    const int4* four = reinterpret_cast<const int4*>(said + first);
#pragma unroll 1
    for (int i0 = tid; i0 < fours; i0 += kAdjustAhead * THREADS) {
      int4 t[kAdjustAhead];                                // loads in flight together (behind one another's atomics they would not be)
#pragma unroll
      for (int k = 0; k < kAdjustAhead; ++k) t[k] = i0 + k * THREADS < fours ? four[i0 + k * THREADS] : make_int4(-1, -1, -1, -1);
#pragma unroll
      for (int k = 0; k < kAdjustAhead; ++k) {
        const int at = first + 4 * (i0 + k * THREADS);
        one(t[k].x, at >= prompt); one(t[k].y, at + 1 >= prompt); one(t[k].z, at + 2 >= prompt); one(t[k].w, at + 3 >= prompt);
      }
    }
    const int rest = first + 4 * fours + tid;
    if (rest < length) one(said[rest], rest >= prompt);
    if (row0 >= 0)
      for (int j = 1 + tid; j < 32 * p.words && j < p.rows - row0; j += THREADS)
        if (p.sees[row * p.lds + (j >> 5)] >> (j & 31) & 1u) one(p.draft[row0 + j], true);
  };
  auto mark = [&](int at, bool) {
    const uint32_t bit = 1u << (at & 31);
    if (marked[at >> 5] & bit) return;                     // (by now, perhaps; then the atomic says so)
    if (atomicOr(marked + (at >> 5), bit) & bit) return;
    table[at] = 0;
  };
  each(mark);
  for (int e = b0 + tid; e < b1; e += THREADS) {
    const int token = p.bias_id[e];
    if (static_cast<unsigned>(token - from) < tokens) mark(token - lo, false);
  }
  const uint32_t* mask = p.mask != nullptr ? p.mask + row * p.ldm : nullptr;
  auto allowed = [&](int token) { return mask == nullptr || (mask[token >> 5] >> (token & 31) & 1u) != 0; };
  if (copies) {
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      const int at = lo + (k * THREADS + tid) * N;
      if (at >= p.vocab || at + N <= 0) continue;
      if (at >= 0 && at + N <= p.vocab) {
        if (mask != nullptr) {
          const uint32_t bits = __funnelshift_r(mask[at >> 5], mask[(at + N - 1) >> 5], at & 31);
          uint32_t* x = &v[k].x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (N == 8) {
              const uint32_t keep = (bits >> (2 * j) & 1u ? 0xFFFFu : 0u) | (bits >> (2 * j + 1) & 1u ? 0xFFFF0000u : 0u);
              x[j] = (x[j] & keep) | (0xFF80FF80u & ~keep);
            } else {
              if (!(bits >> j & 1u)) x[j] = 0xFF800000u;
            }
          }
        }
        if (wide) {
          *reinterpret_cast<uint4*>(out + at) = v[k];
        } else {
          const T* x = reinterpret_cast<const T*>(&v[k]);
#pragma unroll
          for (int j = 0; j < N; ++j) out[at + j] = x[j];
        }
      } else {                                             // the ends of a row
        for (int token = max(at, 0); token < min(at + N, p.vocab); ++token) {
          if (allowed(token)) out[token] = in[token]; else adjust_store(out[token], -INFINITY);
        }
      }
    }
  }
  __syncthreads();
  if (b1 > b0) {
    for (int e = b0 + tid; e < b1; e += THREADS) {
      const int token = p.bias_id[e];
      if (static_cast<unsigned>(token - from) < tokens) atomicMax(table + (token - lo), min(static_cast<uint32_t>(e - b0) + 1u, kAdjustFar));
    }
    __syncthreads();
  }
  {
    // the marked tokens as a list: a thread has a word of marks
    const int lane = tid & 31;
    uint32_t bits = tid < kRange / 32 ? marked[tid] : 0u;
    const int n = __popc(bits);
    int before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    int base = 0;
    if (lane == 31 && before > 0) base = atomicAdd(&listed, before);
    base = __shfl_sync(0xffffffffu, base, 31) + before - n;
    for (; bits != 0 && base < kAdjustList; bits &= bits - 1) list[base++] = static_cast<uint16_t>(32 * tid + __ffs(bits) - 1);
  }
  each([&](int at, bool own) {
    if (own) atomicAdd(table + at, kAdjustOne); else atomicOr(table + at, kAdjustSeen);
  });
  __syncthreads();
  auto adjust = [&](int at) {
    const int token = lo + at;
    if (!allowed(token)) return;
    const uint32_t w = table[at];
    float x = adjust_load(in[token]);
    if (w >= kAdjustSeen) {
      x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
      if (w >= kAdjustOne) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(w / kAdjustOne))), pres);
    }
    if (w & kAdjustFar) {
      int e = b0 + static_cast<int>(w & kAdjustFar) - 1;
      if ((w & kAdjustFar) == kAdjustFar)                  // a list longer than the words can name: its last entry of the token
        for (e = b1 - 1; p.bias_id[e] != token; --e) {}
      x = __fadd_rn(x, p.bias[e]);
    }
    adjust_store(out[token], x);
  };
  if (listed <= kAdjustList) {
    for (int i = tid; i < listed; i += THREADS) adjust(list[i]);
  } else {                                                 // more than there is room for: all marked ones, a word a warp
    for (int i = tid >> 5; i < kRange / 32; i += THREADS / 32)
      if (marked[i] >> (tid & 31) & 1u) adjust(32 * i + (tid & 31));
  }
}

}  // namespace cb

extern "C" int cb_adjust_logits(const CbAdjust* p, void* stream) {
  using namespace cb;
  if (p->rows <= 0) return 0;
  if (p->vocab < 1 || p->vocab > 1 << 20 || p->rows > 65535 || p->most < 0 || p->most >= (1 << 20) - 256) return -10;
  const int size = p->f32 ? 4 : 2, range = kAdjustBytes / size;
  const dim3 grid((p->vocab + 16 / size - 1 + range - 1) / range, p->rows);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -18;
  if (!sms[dev]) {
    int n = 0;
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<int>(e);
    sms[dev] = n;
  }
  if (static_cast<long long>(grid.x) * grid.y <= 2 * sms[dev])
    return static_cast<int>(p->f32 ? launch(adjust_kernel<float, 1024>, grid, dim3(1024), 0, st, *p) : launch(adjust_kernel<__nv_bfloat16, 1024>, grid, dim3(1024), 0, st, *p));
  return static_cast<int>(p->f32 ? launch(adjust_kernel<float, 256>, grid, dim3(256), 0, st, *p) : launch(adjust_kernel<__nv_bfloat16, 256>, grid, dim3(256), 0, st, *p));
}
