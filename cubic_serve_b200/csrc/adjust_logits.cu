// Logits as the requests want them: penalties for repeated tokens, biases of chosen tokens, masks of grammars.
//
// For token t of a row: s = whether the request's prompt or output holds it, c = how often its output does (with the drafts that lead to the row), b its bias:
//   x = logit;  s: x = x > 0 ? x / repetition : x * repetition;  x -= frequency * c;  c > 0: x -= presence;  x += b;  not allowed: x = -inf
// in fp32, rounded once to the type of the logits.
//
// A block has a range of a row's tokens and a word for each of them in shared memory: it reads the request's history, counts the tokens of its range and
// then passes over the range once.
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
  int rows, vocab, n, most, biases, words, f32, chunk;
};

namespace cb {

// A token's word: index of its bias + 1 (kAdjustFar: at least that), seen, count
static constexpr uint32_t kAdjustFar = 2047u, kAdjustSeen = 1u << 11, kAdjustOne = 1u << 12;
static constexpr int kAdjustThreads = 512;

template <typename T>
__device__ __forceinline__ float adjust_load(const T* p);
template <>
__device__ __forceinline__ float adjust_load(const float* p) { return *p; }
template <>
__device__ __forceinline__ float adjust_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void adjust_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void adjust_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

template <typename T>
__global__ void __launch_bounds__(kAdjustThreads)
adjust_kernel(const CbAdjust p) {
  extern __shared__ uint32_t table[];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, tid = threadIdx.x, lo = blockIdx.x * p.chunk, size = min(p.chunk, p.vocab - lo);
  const int r = p.request != nullptr ? p.request[row] : row;
  const bool known = r >= 0 && r < p.n;
  for (int i = tid; i < size; i += kAdjustThreads) table[i] = 0;
  __syncthreads();
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int b0 = 0, b1 = 0;
  if (known) {
    if (p.repetition != nullptr) rep = p.repetition[r];
    if (p.frequency != nullptr) freq = p.frequency[r];
    if (p.presence != nullptr) pres = p.presence[r];
    if (p.bias_at != nullptr) {
      b0 = max(p.bias_at[r], 0);
      b1 = min(p.bias_at[r + 1], p.biases);
      for (int e = b0 + tid; e < b1; e += kAdjustThreads) {
        const unsigned at = p.bias_id[e] - lo;
        if (at < static_cast<unsigned>(size)) atomicMax(table + at, min(static_cast<uint32_t>(e - b0) + 1u, kAdjustFar));
      }
      __syncthreads();
    }
    const int length = min(max(p.length[r], 0), p.most), prompt = p.prompt != nullptr ? p.prompt[r] : 0;
    const int* said = p.history + r * p.ldh;
    for (int i = tid; i < length; i += kAdjustThreads) {
      const unsigned at = said[i] - lo;
      if (at >= static_cast<unsigned>(size)) continue;
      if (i < prompt) atomicOr(table + at, kAdjustSeen); else atomicAdd(table + at, kAdjustOne);
    }
    if (p.draft != nullptr) {
      const int first = p.row0[r];
      for (int j = 1 + tid; j < 32 * p.words; j += kAdjustThreads) {
        if (!(p.sees[row * p.lds + (j >> 5)] >> (j & 31) & 1u) || first < 0 || first + j >= p.rows) continue;
        const unsigned at = p.draft[first + j] - lo;
        if (at < static_cast<unsigned>(size)) atomicAdd(table + at, kAdjustOne);
      }
    }
  }
  __syncthreads();
  const T* in = static_cast<const T*>(p.logits) + row * p.ldl + lo;
  T* out = static_cast<T*>(p.out) + row * p.ldo + lo;
  const uint32_t* mask = p.mask != nullptr ? p.mask + row * p.ldm : nullptr;
  for (int i = tid; i < size; i += kAdjustThreads) {
    const uint32_t w = table[i];
    float x = adjust_load(in + i);
    if (w >= kAdjustSeen) {
      x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
      if (w >= kAdjustOne) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(w / kAdjustOne))), pres);
    }
    if (w & kAdjustFar) {
      int e = b0 + static_cast<int>(w & kAdjustFar) - 1;
      if ((w & kAdjustFar) == kAdjustFar)
        for (e = b1 - 1; p.bias_id[e] != lo + i; --e) {}
      x = __fadd_rn(x, p.bias[e]);
    }
    if (mask != nullptr && !(mask[(lo + i) >> 5] >> ((lo + i) & 31) & 1u)) x = -INFINITY;
    adjust_store(out + i, x);
  }
}

}  // namespace cb

extern "C" int cb_adjust_logits(const CbAdjust* p, void* stream) {
  using namespace cb;
  if (p->rows <= 0) return 0;
  if (p->vocab < 1 || p->rows > 65535 || p->most < 0 || p->most >= (1 << 20) - 256) return -10;
  CbAdjust a = *p;
  a.chunk = 8192;
  const dim3 grid((p->vocab + a.chunk - 1) / a.chunk, p->rows);
  const size_t smem = static_cast<size_t>(a.chunk) * 4;
  auto k = p->f32 ? adjust_kernel<float> : adjust_kernel<__nv_bfloat16>;
  return static_cast<int>(launch(k, grid, dim3(kAdjustThreads), smem, static_cast<cudaStream_t>(stream), a));
}
