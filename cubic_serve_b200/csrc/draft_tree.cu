// The end of a round of drafts in a tree: the path that the target agrees with, and its keys and values behind the context.
//
// verify_tree: from node 0 on, the target's choice at a node is emitted; the first child that holds it is the next node, and without one the walk ends.
// keep_tokens: the nodes of a path, path[0] = 0 < path[1] < .., lie at the slots start + path[k] of their request; line start + path[k] of every layer and
// key / value head becomes line start + k.  path[k] >= k, so a line is read before anything is put in its place: a warp
// loads four lines, puts them down and goes on.  A lane has four channels, and no other lane the words that hold them (K words of 4 bits: lanes t and t + 4 exchange their halves).
//
// Bound by latency, a few dependent trips to memory each: a warp walks a request's tree, 32 nodes a look; a warp moves the lines of a request, layer and head, so that
// these fill the GPU.  Both together for a tree of 8 nodes and 36 layers 5.0 us, for 64 of 26 nodes and 12 layers 8.2, for 256 of 16 nodes 11.6.
#include "paged_attn.cuh"

// Packed by ops/native.py::VERIFY_TREE.
struct CbVerifyTree {
  const int* target;         // [rows] the target's choice behind every node
  const int* tokens;         // [rows] the nodes' tokens (node 0: any)
  const int* parents;        // [rows] node that a node follows, -1 for node 0
  const int* row0;           // [n] first row of the request
  const int* count;          // [n] nodes
  int* accepted;             // [n] drafts on the path
  int* path;                 // [n, depth] nodes of the path, -1 behind it
  int* emitted;              // [n, depth] the target's choices along the path, -1 behind them
  int n, rows, depth;
};

// Packed by ops/native.py::KEEP_TOKENS.
struct CbKeepTokens {
  const unsigned long long* caches;   // [layers] addresses of [pages][Hkv][blob]
  const int* table;                   // [table_rows, width], row stride ld
  const int* request;                 // [n] row of the block table
  const int* start;                   // [n] slots before node 0
  const int* accepted;                // [n]
  const int* path;                    // [n, depth], row stride ldp
  uint32_t* status;
  long long ld, ldp;
  int n, layers, Hkv, pages, table_rows, width, depth, k_bits, v_bits;
};

namespace cb {

__global__ void __launch_bounds__(128)
verify_tree_kernel(const CbVerifyTree p) {
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= p.n) return;
  const int row0 = p.row0[i];
  const int count = row0 >= 0 && row0 < p.rows ? min(p.count[i], p.rows - row0) : 0;
  int* path = p.path + static_cast<size_t>(i) * p.depth;
  int* emitted = p.emitted + static_cast<size_t>(i) * p.depth;
  int cur = 0, len = 0;
  while (len < p.depth && cur < count) {
    const int want = p.target[row0 + cur];
    if (lane == 0) { path[len] = cur; emitted[len] = want; }
    ++len;
    int next = count;
    for (int j0 = cur + 1; j0 < count && next == count; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t fits = __ballot_sync(0xffffffffu, j < count && p.parents[row0 + j] == cur && p.tokens[row0 + j] == want);
      if (fits) next = j0 + __ffs(fits) - 1;
    }
    cur = next;
  }
  for (int k = len + lane; k < p.depth; k += 32) path[k] = emitted[k] = -1;
  if (lane == 0) p.accepted[i] = max(len - 1, 0);
}

// A lane's codes of a token, as pf_codes_k / pf_codes_v read them, into the page.
template <int BITS>
__device__ __forceinline__ void put_codes_k(uint8_t* k, int tok, int lane, uint32_t codes) {
  if constexpr (BITS == 8) {
    *reinterpret_cast<uint32_t*>(k + (lane >> 2) * 256 + tok * 16 + (lane & 3) * 4) = codes;
  } else {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 4);
    if (lane & 4) return;
    const int blk = lane >> 3, t = lane & 3;
    *reinterpret_cast<uint32_t*>(k + blk * 256 + tok * 16 + t * 4) = (codes & 0x0F0F0F0Fu) | (other & 0x0F0F0F0Fu) << 4;
    if constexpr (BITS == 6) {
      uint32_t* at = reinterpret_cast<uint32_t*>(k + kPageTokens * kD / 2 + blk * 128 + (tok & 7) * 16 + t * 4);
      const uint32_t high = (codes & 0x30303030u) | (other & 0x30303030u) << 2;        // bits 4..7 of every byte
      *at = tok < 8 ? (*at & 0x0F0F0F0Fu) | high : (*at & 0xF0F0F0F0u) | high >> 4;
    }
  }
}
template <int BITS>
__device__ __forceinline__ void put_codes_v(uint8_t* v, int tok, int lane, uint32_t codes) {
  const int pair = tok >> 1, odd = tok & 1, at = lane ^ ((pair & 3) << 2);
  if constexpr (BITS == 8) {
    uint2* w = reinterpret_cast<uint2*>(v + pair * 256 + at * 8);
    uint2 x = *w;
    x.x = odd ? prmt(x.x, codes, 0x5240u) : prmt(x.x, codes, 0x3514u);                 // bytes 1 and 3, or 0 and 2
    x.y = odd ? prmt(x.y, codes, 0x7260u) : prmt(x.y, codes, 0x3716u);
    *w = x;
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(v + pair * 128 + at * 4);
    *w = odd ? (*w & 0x0F0F0F0Fu) | (codes & 0x0F0F0F0Fu) << 4 : (*w & 0xF0F0F0F0u) | (codes & 0x0F0F0F0Fu);
    if constexpr (BITS == 6) {
      uint32_t* h = reinterpret_cast<uint32_t*>(v + kPageTokens * kD / 2 + (pair & 3) * 128 + at * 4);
      const int shift = (pair < 4 ? 4 : 0) + 2 * odd;                                  // where bit 0 of the two high bits goes
      *h = (*h & ~(0x03030303u << shift)) | ((codes >> 4) & 0x03030303u) << shift;
    }
  }
}

template <int KBITS, int VBITS>
__global__ void __launch_bounds__(256)
keep_tokens_kernel(const CbKeepTokens p, const KvLayout lay) {
  constexpr int kLines = 4;
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x, lane = threadIdx.x & 31, unit = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (unit >= p.layers * p.Hkv) return;
  const int accepted = p.accepted[i], slot = p.request[i], start = p.start[i];
  if (accepted <= 0) return;
  const int* path = p.path + i * p.ldp;
  bool bad = accepted >= p.depth || slot < 0 || slot >= p.table_rows || start < 0;
  if (!bad) {
    const int layer = unit / p.Hkv, head = unit - layer * p.Hkv;
    uint8_t* cache = reinterpret_cast<uint8_t*>(p.caches[layer]);
    const int* table = p.table + slot * p.ld;
    auto page_of = [&](int t) {                          // -1: not there
      const int at = t / kPageTokens, page = at < p.width ? table[at] : -1;
      return page < p.pages ? page : -1;
    };
    // a lane has a place of the path, and the pages of its line; the whole path is looked at before any line moves: it rises, and all its pages are there
    int mine = 0, from_page = -1, to_page = -1;
    auto look = [&](int k) {
      if (k > accepted) return;
      mine = path[k];
      bad = bad || mine <= (k > 1 ? path[k - 1] : 0) || mine > (1 << 30) - start;
      if (bad || mine == k) return;
      from_page = page_of(start + mine);
      to_page = page_of(start + k);
      bad = from_page < 0 || to_page < 0;
    };
    for (int k0 = 1; k0 <= accepted; k0 += 32) look(k0 + lane);
    bad = __any_sync(0xffffffffu, bad);
    auto blob = [&](int page) { return cache + (static_cast<size_t>(page) * p.Hkv + head) * lay.blob_bytes; };
    for (int k0 = 1; k0 <= accepted && !bad; k0 += kLines) {
      if (accepted > 32 && k0 % 32 == 1) look(k0 + lane);
      uint32_t kc[kLines], vc[kLines];
      float ks[kLines], vs[kLines];
      uint8_t* to[kLines];
      int tok[kLines];
#pragma unroll
      for (int l = 0; l < kLines; ++l) {
        const int k = k0 + l, of = (k - 1) & 31, at = __shfl_sync(0xffffffffu, mine, of), fp = __shfl_sync(0xffffffffu, from_page, of), tp = __shfl_sync(0xffffffffu, to_page, of);
        to[l] = nullptr;
        if (k > accepted || at == k) continue;
        const uint8_t* from = blob(fp);
        to[l] = blob(tp);
        const int src = (start + at) % kPageTokens;
        tok[l] = (start + k) % kPageTokens;
        kc[l] = pf_codes_k<KBITS>(from, src, lane);
        vc[l] = pf_codes_v<VBITS>(from + lay.v_code_off, src, lane);
        ks[l] = *reinterpret_cast<const float*>(from + lay.k_scale_off + src * 16 + (lane >> 3) * 4);
        vs[l] = *reinterpret_cast<const float*>(from + lay.v_scale_off + src * 16 + (lane >> 3) * 4);
      }
      __syncwarp();
#pragma unroll
      for (int l = 0; l < kLines; ++l) {
        if (to[l] == nullptr) continue;                  // (the same for all lanes)
        put_codes_k<KBITS>(to[l], tok[l], lane, kc[l]);
        put_codes_v<VBITS>(to[l] + lay.v_code_off, tok[l], lane, vc[l]);
        if ((lane & 7) == 0) {
          *reinterpret_cast<float*>(to[l] + lay.k_scale_off + tok[l] * 16 + (lane >> 3) * 4) = ks[l];
          *reinterpret_cast<float*>(to[l] + lay.v_scale_off + tok[l] * 16 + (lane >> 3) * 4) = vs[l];
        }
      }
      __syncwarp();
    }
  }
  if (bad && lane == 0) atomicExch(p.status, static_cast<uint32_t>(kErrBadArgument));
}

}  // namespace cb

extern "C" {

int cb_verify_tree(const CbVerifyTree* p, void* stream) {
  using namespace cb;
  if (p->n <= 0) return 0;
  if (p->depth < 1) return -10;
  return static_cast<int>(launch(verify_tree_kernel, dim3((p->n + 3) / 4), dim3(128), 0, static_cast<cudaStream_t>(stream), *p));
}

int cb_keep_tokens(const CbKeepTokens* p, void* stream) {
  using namespace cb;
  if (p->n <= 0 || p->layers <= 0) return 0;
  if (p->Hkv <= 0 || p->depth < 1 || (p->layers * static_cast<long long>(p->Hkv) + 7) / 8 > 65535) return -10;
  const KvLayout lay = make_kv_layout(kD, p->k_bits, p->v_bits);
  return with_kv_bits(p->k_bits, p->v_bits, [&](auto kb, auto vb) {
    return static_cast<int>(launch(keep_tokens_kernel<decltype(kb)::value, decltype(vb)::value>, dim3(p->n, (p->layers * p->Hkv + 7) / 8), dim3(256), 0,
                                   static_cast<cudaStream_t>(stream), *p, lay));
  });
}

}  // extern "C"
