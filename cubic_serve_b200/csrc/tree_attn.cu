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

// One row over the tokens [lo, hi) in fp32, by a warp whose lanes have four channels each.  `sees`: the row's words.
template <int KBITS, int VBITS>
__device__ __forceinline__ void tree_row(const CbTreeAttn& p, const KvLayout& lay, const TreeRequest& r, int kvh, int lo, int hi, const uint32_t* sees, const __nv_bfloat16* q,
                                         int lane, float& m, float& sum, float (&o)[4], bool& bad) {
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
    const uint8_t* blob = p.cache + (static_cast<size_t>(page) * p.Hkv + kvh) * lay.blob_bytes;
    const uint32_t kc = pf_codes_k<KBITS>(blob, tok, lane), vc = pf_codes_v<VBITS>(blob + lay.v_code_off, tok, lane);
    const float ks = *reinterpret_cast<const float*>(blob + lay.k_scale_off + tok * 16 + (lane >> 3) * 4);
    const float vs = *reinterpret_cast<const float*>(blob + lay.v_scale_off + tok * 16 + (lane >> 3) * 4);
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

template <int KBITS, int VBITS>
__global__ void __launch_bounds__(256)
tree_simple_kernel(const CbTreeAttn p, const KvLayout lay) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, kvh = blockIdx.y, G = p.Hq / p.Hkv;
  bool bad = false;
  const TreeRequest r = tree_request(p, blockIdx.x, bad);
  for (int row = blockIdx.z * 8 + (threadIdx.x >> 5); row < r.count * G; row += gridDim.z * 8) {
    const int node = row / G, at = (kvh * G + row - node * G) * kD;
    float m, sum, o[4];
    tree_row<KBITS, VBITS>(p, lay, r, kvh, 0, r.total, p.masks + (r.row0 + node) * p.ldm, p.q + (r.row0 + node) * p.ldq + at, lane, m, sum, o, bad);
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;                  // NaN stays
    reinterpret_cast<uint2*>(p.out + (r.row0 + node) * p.ldo + at)[lane] = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  }
  if (bad && lane == 0) atomicExch(p.status, static_cast<uint32_t>(kErrBadArgument));
}

}  // namespace cb

extern "C" int cb_tree_attn(const CbTreeAttn* p, void* stream) {
  using namespace cb;
  if (p->n <= 0) return 0;
  if (p->n > kTreeMaxRequests || p->words < 1 || p->words > kTreeMaxWords || p->Hkv <= 0 || p->Hq % p->Hkv != 0 || p->Hq / p->Hkv > kTreeMaxGroup || p->width > 1 << 26) return -10;
  const KvLayout lay = make_kv_layout(kD, p->k_bits, p->v_bits);
  return with_kv_bits(p->k_bits, p->v_bits, [&](auto kb, auto vb) {
    return static_cast<int>(launch(tree_simple_kernel<decltype(kb)::value, decltype(vb)::value>, dim3(p->n, p->Hkv, 8), dim3(256), 0, static_cast<cudaStream_t>(stream), *p, lay));
  });
}
