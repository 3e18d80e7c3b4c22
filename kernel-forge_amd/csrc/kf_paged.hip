// The paged KV cache around its attention: the tables of a step from the requests' lengths, and the writer that rotates q
// and k and puts k and v into their slots.
#include <algorithm>

#include "kf_attn_tiles.h"
#include "kf_launch.h"

namespace kf {
namespace {

// ---- tables ---------------------------------------------------------------------------------------------
// Request r holds ceil(context / block) pages and needs ceil((context + new) / block).  The new pages of all requests, in
// order, come from the top of the stack of free pages; its tokens follow those of the requests before it.  Both
// need sums over the requests before: every workgroup adds them up for its own request (4 bytes each, from L2), which
// costs less than a second launch would.  Bound by latency: a load, a sum in the workgroup, the writes.  Workgroup (r, y)
// writes request r's share y of the tokens; r = seqs the totals and the rows behind the last token.
constexpr int kTablesThreads = 256;

struct Lens {
  int context, fresh_from, fresh;  // tokens cached; first new page and how many
  int tokens;
};
__device__ __forceinline__ Lens request_lens(const TablesArgs& a, int r) {
  const int64_t cap = (int64_t)a.width << a.log2_block;
  const int64_t context = max(load_const(a.context_lens, r), 0), tokens = max(load_const(a.new_lens, r), 0);
  const int block = (1 << a.log2_block) - 1;
  // Pages past the table's width are not taken.
  const int held = (int)((min(context, cap) + block) >> a.log2_block);
  const int need = (int)((min(context + tokens, cap) + block) >> a.log2_block);
  return Lens{(int)context, held, need - held, (int)tokens};
}

__global__ __launch_bounds__(kTablesThreads) void paged_tables_kernel(TablesArgs a) {
  __shared__ int64_t parts[2][kTablesThreads / 64];
  const int r = blockIdx.x, tid = threadIdx.x;
  int64_t tokens = 0, pages = 0;  // 64 bits: no lengths make the sums wrap into indexes
  for (int i = tid; i < r; i += kTablesThreads) {
    const Lens l = request_lens(a, i);
    tokens += l.tokens;
    pages += l.fresh;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    tokens += __shfl_xor(tokens, off);
    pages += __shfl_xor(pages, off);
  }
  if ((tid & 63) == 0) {
    parts[0][tid >> 6] = tokens;
    parts[1][tid >> 6] = pages;
  }
  __syncthreads();
  tokens = pages = 0;
#pragma unroll
  for (int w = 0; w < kTablesThreads / 64; ++w) {
    tokens += parts[0][w];
    pages += parts[1][w];
  }

  const int count = min(max(load_const(a.free_count, 0), 0), a.free_capacity);
  const int first = blockIdx.y * kTablesThreads + tid, step = gridDim.y * kTablesThreads;
  if (r == a.seqs) {
    if (first == 0) {
      a.cu_new[r] = (int)min(tokens, (int64_t)0x7fffffff);
      *a.free_left = (int)max(count - pages, (int64_t)0);
    }
    for (int64_t i = tokens + first; i < a.max_tokens; i += step) a.positions[i] = a.slots[i] = -1;
    return;
  }
  const Lens l = request_lens(a, r);
  if (first == 0) {
    a.cu_new[r] = (int)min(tokens, (int64_t)0x7fffffff);
    a.seq_lens[r] = (int)min((int64_t)l.context + l.tokens, (int64_t)0x7fffffff);
  }
  int* const row = a.table + (int64_t)r * a.table_stride;
  auto new_page = [&](int j) {  // the request's j-th new page, -1 when the stack is empty
    const int64_t at = count - 1 - pages - j;
    return at >= 0 ? a.free_pages[at] : -1;
  };
  for (int j = first; j < l.fresh; j += step) row[l.fresh_from + j] = new_page(j);
  const int mask = (1 << a.log2_block) - 1;
  for (int64_t i = first; i < l.tokens && tokens + i < a.max_tokens; i += step) {
    const int64_t pos = l.context + i;
    const int64_t p = pos >> a.log2_block;
    const int page = p >= a.width ? -1 : p >= l.fresh_from ? new_page((int)p - l.fresh_from) : row[p];
    a.positions[tokens + i] = pos;
    a.slots[tokens + i] = page < 0 ? -1 : ((int64_t)page << a.log2_block) + (pos & mask);
  }
}

// ---- RoPE and the cache ------------------------------------------------------------------------------------
// y[j] = x[j] cos[p, j] + x[(j + d / 2) mod d] sin[p, j] in 32 bits, rounded once; v as it is.  Bound by memory: one thread
// takes a piece of V values and the piece d / 2 further, which rotate into each other, of one head of one token, so every
// value is read once and written once (k twice: beside q for attention straight from the projection, and into its slot).
template <class E, int V>
__global__ __launch_bounds__(256) void rope_paged_kernel(RopePagedArgs a, uint32_t pieces, uint32_t items) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= items) return;
  const uint32_t heads = a.heads + 2 * a.kv_heads, per_token = heads * pieces;
  const uint32_t t = i / per_token, h = (i - t * per_token) / pieces, c = i - t * per_token - h * pieces;
  const int d = a.head_dim, half = d / 2;
  typedef uint32_t vec_t __attribute__((ext_vector_type(V / 2)));
  const E* const src = (const E*)a.qkv + (int64_t)t * a.qkv_stride + (int64_t)h * d + c * V;
  vec_t x0 = *(const vec_t*)src, x1 = *(const vec_t*)(src + half);
  const int64_t pos = a.positions[t];
  const bool inside = pos >= 0 && pos < a.max_pos;
  if ((int)h < a.heads + a.kv_heads) {
    const float* const cos = (const float*)a.cos + (inside ? pos : 0) * d + c * V;
    const float* const sin = (const float*)a.sin + (inside ? pos : 0) * d + c * V;
    vec_t y0, y1;
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const float a0 = Elem<E>::lo(x0[e]), a1 = Elem<E>::hi(x0[e]), b0 = Elem<E>::lo(x1[e]), b1 = Elem<E>::hi(x1[e]);
      y0[e] = Elem<E>::pack(fmaf(b0, sin[2 * e], a0 * cos[2 * e]), fmaf(b1, sin[2 * e + 1], a1 * cos[2 * e + 1]));
      y1[e] = Elem<E>::pack(fmaf(a0, sin[half + 2 * e], b0 * cos[half + 2 * e]),
                            fmaf(a1, sin[half + 2 * e + 1], b1 * cos[half + 2 * e + 1]));
    }
    x0 = y0;
    x1 = y1;
    E* const out = (E*)a.qk + ((int64_t)t * (a.heads + a.kv_heads) + h) * d + c * V;
    *(vec_t*)out = x0;
    *(vec_t*)(out + half) = x1;
    if ((int)h < a.heads) return;
  }
  const int64_t slot = a.slots[t];
  if (!inside || slot < 0 || slot >= a.num_slots) return;
  const int64_t page = slot >> a.log2_block, in_page = slot & ((1 << a.log2_block) - 1);
  const bool is_v = (int)h >= a.heads + a.kv_heads;
  const int64_t kv = h - a.heads - (is_v ? a.kv_heads : 0);
  E* const dst = is_v ? (E*)a.cache_v + page * a.v_page + kv * a.v_head + in_page * a.v_token + c * V
                      : (E*)a.cache_k + page * a.k_page + kv * a.k_head + in_page * a.k_token + c * V;
  *(vec_t*)dst = x0;
  *(vec_t*)(dst + half) = x1;
}

template <class E>
hipError_t rope_launch(const RopePagedArgs& a, hipStream_t stream) {
  const int v = a.head_dim % 16 == 0 ? 8 : 4;  // 16-byte pieces where half a head is whole pieces
  const uint32_t pieces = a.head_dim / 2 / v;
  const uint32_t items = (uint32_t)a.tokens * (uint32_t)(a.heads + 2 * a.kv_heads) * pieces;
  const dim3 grid((items + 255) / 256);
  if (v == 8) rope_paged_kernel<E, 8><<<grid, 256, 0, stream>>>(a, pieces, items);
  else rope_paged_kernel<E, 4><<<grid, 256, 0, stream>>>(a, pieces, items);
  return hipGetLastError();
}

}  // namespace

hipError_t paged_tables_launch(const TablesArgs& a, hipStream_t stream) {
  // About 1,024 tokens per workgroup where there are few requests; one workgroup each where there are many.
  const int64_t shares = std::min<int64_t>(((int64_t)a.max_tokens + 1023) / 1024, std::max(1, 1024 / (a.seqs + 1)));
  paged_tables_kernel<<<dim3(a.seqs + 1, (unsigned)std::max<int64_t>(shares, 1)), kTablesThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t rope_paged_launch(const RopePagedArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? rope_launch<bhalf_t>(a, stream) : rope_launch<half_t>(a, stream);
}

}  // namespace kf
