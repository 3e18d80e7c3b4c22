// Decoding with drafted tokens over the paged cache: the tables of the drafts' trees, their verification, and what is kept of
// them in the cache.  (Their attention: kf_few_rows.h, kf_flash.hip.)
//
// A request's new tokens are the nodes of a tree: node 0 is its pending token, the parent of another node is one of a smaller
// number.  A request has 64 nodes at most, so a set of nodes is a 64-bit word and a wavefront has a lane for each.
#include <algorithm>

#include "kf_attn_tiles.h"
#include "kf_launch.h"

namespace kf {
namespace {

constexpr int kNodes = 64;

// A request's tree, lane i its node i.
struct Tree {
  int first, len, nodes;  // its first row, its new tokens, those of them that are nodes
  int parent;             // of this lane's node; -1: none, or not a node
  uint64_t ancestors;     // and the node itself
};
__device__ __forceinline__ Tree load_tree(const int* parents, const int* cu, int r, int seqs, int tokens, int most, int lane) {
  Tree t;
  t.first = seq_offset(cu, r, seqs, tokens);
  t.len = max(seq_offset(cu, r + 1, seqs, tokens) - t.first, 0);
  t.nodes = min(t.len, most);
  const int p = lane < t.nodes ? parents[t.first + lane] : -1;
  t.parent = (unsigned)p < (unsigned)lane ? p : -1;
  // Pointers doubled: after n rounds a node knows 2^n - 1 ancestors and where the next one is.  A root points to itself.
  t.ancestors = 1ull << lane;
  int jump = t.parent < 0 ? lane : t.parent;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    t.ancestors |= __shfl(t.ancestors, jump);
    jump = __shfl(jump, jump);
  }
  return t;
}

// A lane's value, the lane the same for all.  As with all exchange of lanes here: asked for by all of them, outside of branches,
// as a lane that has not come there has nothing to give.
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
template <class T>
__device__ __forceinline__ T of_lane(T v, int lane) {
  static_assert(sizeof(T) == 8, "two words");
  const u32x2 w = bit_cast<u32x2>(v);
  return bit_cast<T>(u32x2{(uint32_t)of_lane((int)w[0], lane), (uint32_t)of_lane((int)w[1], lane)});
}

// ---- tables ---------------------------------------------------------------------------------------------
// A wavefront per request.  Bound by latency: the offsets, then the parents, then six rounds of lane exchange.
constexpr int kTreeWaves = 4;

__global__ __launch_bounds__(64 * kTreeWaves) void draft_trees_kernel(DraftTreesArgs a) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * kTreeWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r < a.seqs) {
    const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens, kNodes, lane);
    const int64_t context = (int64_t)load_const(a.seq_lens, r) - t.len;
    for (int i = lane; i < t.len; i += 64) {  // past the 64th: no node
      a.ancestors[t.first + i] = i < kNodes ? t.ancestors : 0;
      a.positions[t.first + i] = i < kNodes ? context + __popcll(t.ancestors) - 1 : -1;
    }
  }
  // Rows in no request.
  for (int64_t i = seq_offset(a.cu, a.seqs, a.seqs, a.tokens) + (int64_t)blockIdx.x * 64 * kTreeWaves + threadIdx.x;
       i < a.tokens; i += (int64_t)gridDim.x * 64 * kTreeWaves) {
    a.ancestors[i] = 0;
    a.positions[i] = -1;
  }
}

// ---- verification: what all forms share ---------------------------------------------------------------------
// A node's child is accepted or not by itself and its elder siblings; the path is the nodes all of whose ancestors are the
// first accepted child of their parents.  So no walk from node to node: every lane judges its own node, and one bit test per node
// gives the path.

// Of accepted children with one parent the first.
__device__ __forceinline__ bool first_accepted(bool accepted, int parent, int lane) {
  bool first = accepted;
  for (uint64_t m = __ballot(accepted); m; m &= m - 1) {
    const int e = __builtin_ctzll(m), same = of_lane(parent, e);
    first &= !(lane > e && parent == same);
  }
  return first;
}
// The nodes on the path, node 0 (which is given) among them; a chain from it.
__device__ __forceinline__ uint64_t path_of(const Tree& t, bool chosen, int lane) {
  const uint64_t ok = __ballot(chosen) | 1;
  return __ballot(lane < t.nodes && (t.ancestors & ~ok) == 0);
}
// counts, path and emitted tokens of request r but for the token behind the path; last: the path's last node.
__device__ __forceinline__ void write_path(const VerifyArgs& a, int r, const Tree& t, uint64_t on, int64_t token, int lane) {
  const int count = __popcll(on), rank = __popcll(on & ((1ull << lane) - 1));
  int* const path = a.path + (int64_t)r * a.width;
  int64_t* const emitted = a.emitted + (int64_t)r * a.width;
  if (lane == 0) a.counts[r] = count;
  if (on >> lane & 1) {
    path[rank] = lane;
    if (rank > 0) emitted[rank - 1] = token;
  }
  if (lane >= count && lane < a.width) {
    path[lane] = -1;
    emitted[lane] = -1;
  }
}

// ---- by the largest score -----------------------------------------------------------------------------------
// The largest of a row as a 64-bit key: the value's order in the upper half (NaN above all numbers), the index's reverse in the
// lower, so that of equal values the first wins.
__device__ __forceinline__ uint64_t score_key(float x, int index) {
  const uint32_t b = bit_cast<uint32_t>(x + 0.0f);  // -0 is 0
  const uint32_t order = x != x ? 0xFFFFFFFFu : b >> 31 ? ~b : b | 0x80000000u;
  return (uint64_t)order << 32 | (0xFFFFFFFFu - (uint32_t)index);
}

// Eight values of a row from any 4-byte boundary on.  (16-byte loads from addresses between two words read others.)
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  typedef uint32_t vec_t __attribute__((ext_vector_type(4), aligned(4)));
  const u32x4 v = *(const vec_t*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Elem<T>::lo(v[i]);
    x[2 * i + 1] = Elem<T>::hi(v[i]);
  }
}
typedef float row4_t __attribute__((ext_vector_type(4), aligned(4)));
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const row4_t v = *(const row4_t*)p, w = *(const row4_t*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = v[i];
    x[4 + i] = w[i];
  }
}

constexpr int kBestThreads = 256, kBestStep = 8 * kBestThreads;

// keys[row * shares + share] = the largest of the share's part of the row.
template <class T>
__global__ __launch_bounds__(kBestThreads) void best_token_kernel(VerifyArgs a, int shares, int part) {
  __shared__ uint64_t keys[kBestThreads / 64];
  const int row = blockIdx.x / shares, share = blockIdx.x - row * shares;
  if (row >= seq_offset(a.cu, a.seqs, a.seqs, a.tokens_count)) return;
  const T* const src = (const T*)a.target + (int64_t)row * a.target_row;
  const int begin = share * part, end = min(begin + part, a.vocab), tid = threadIdx.x;
  float best = -__builtin_inff();
  int at = 0;
  bool any = false;  // a row of -inf has its first index as well
  auto take = [&](float x, int i) {
    if (!any || x > best || (x != x && best == best)) {
      best = x;
      at = i;
      any = true;
    }
  };
  // A row of 16-bit values may begin between two words: its first value is taken alone.
  const int odd = sizeof(T) == 2 ? (int)((uintptr_t)(src + begin) >> 1 & 1) : 0;
  if (odd && tid == 0 && begin < end) take((float)src[begin], begin);
  int i = begin + odd + 8 * tid;
  for (; i + 8 <= end; i += kBestStep) {
    float x[8];
    load8(src + i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) take(x[e], i + e);
  }
  for (int e = 0; e < 8 && i + e < end; ++e) take((float)src[i + e], i + e);
  uint64_t key = any ? score_key(best, at) : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t other = __shfl_xor(key, off);
    key = other > key ? other : key;
  }
  if ((tid & 63) == 0) keys[tid >> 6] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kBestThreads / 64; ++w) key = keys[w] > key ? keys[w] : key;
    static_cast<uint64_t*>(a.ws)[blockIdx.x] = key;
  }
}

__global__ __launch_bounds__(64 * kTreeWaves) void verify_best_kernel(VerifyArgs a, int shares) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * kTreeWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= a.seqs) return;
  const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens_count, a.width, lane);
  int64_t token = -1, best = -1;
  if (lane < t.nodes) {
    const uint64_t* const keys = static_cast<const uint64_t*>(a.ws) + (int64_t)(t.first + lane) * shares;
    token = a.tokens[t.first + lane];
    uint64_t key = 0;
    for (int s = 0; s < shares; ++s) key = keys[s] > key ? keys[s] : key;
    best = 0xFFFFFFFFu - (uint32_t)key;
  }
  const int64_t wanted = __shfl(best, max(t.parent, 0));
  const bool accepted = t.parent >= 0 && token == wanted;
  const uint64_t on = path_of(t, first_accepted(accepted, t.parent, lane), lane);
  write_path(a, r, t, on, token, lane);
  const int last = on ? 63 - __clzll((long long)on) : -1;
  if (lane == last) a.emitted[(int64_t)r * a.width + __popcll(on) - 1] = best;
}

// ---- from probabilities and given random numbers -------------------------------------------------------------
// What is left of row t's mass after its rejected children is f = max(p - a q, 0) where they were drawn from q, f = p without their
// tokens where they were given.  One launch adds f up over pieces of the path's last row, the next finds the piece and the
// token at which the running sum passes u times all of it.  In 64 bits, as an index is an integer and 32 bits would move it.
constexpr int kPickThreads = 256, kPiece = 16 * kPickThreads;  // values of a row

struct Last {  // of a request's path
  double a;      // how much of the draft's probabilities is taken off
  int row;       // of target and draft; -1: the request has no new tokens
  int node;
};
struct VerifySpace {
  double* sums;       // [seqs, pieces]
  Last* last;         // [seqs]
  double* taken;      // drawn: [tokens] a of every row all of whose children are rejected
  int* chosen;        // drawn: [tokens] 1: the first accepted child of its parent
};
__device__ __host__ inline VerifySpace verify_space(void* ws, int seqs, int pieces, int tokens) {
  VerifySpace s;
  s.sums = static_cast<double*>(ws);
  s.last = reinterpret_cast<Last*>(s.sums + (size_t)seqs * pieces);
  s.taken = reinterpret_cast<double*>(s.last + seqs);
  s.chosen = reinterpret_cast<int*>(s.taken + tokens);
  return s;
}

__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }  // of NaN: nothing

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
// Of a workgroup, the same in all threads.
template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double* parts) {
  v = wave_sum(v);
  __syncthreads();  // the last sum's have been read
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += parts[w];
  return v;
}

// Value i of a row as a double, or 0 for one that is none.
__device__ __forceinline__ double prob_at(const float* row, int64_t token, int vocab) {
  return token >= 0 && token < vocab ? (double)row[token] : 0.0;
}

// Drafts that were drawn from given probabilities, one workgroup per node: which of its children is accepted.  A test after a
// rejection needs a sum over the node's row, so only nodes that the path may still come to make any: children whose first
// test fails end the ways through them, those of a second test keep theirs open.
constexpr int kChooseThreads = 512;
__global__ __launch_bounds__(kChooseThreads) void choose_child_kernel(VerifyArgs a, int pieces) {
  __shared__ double parts[kChooseThreads / 64];
  const int lane = threadIdx.x & 63, node = blockIdx.x, r = blockIdx.y;
  const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens_count, a.width, lane);
  if (node >= t.nodes) return;
  const VerifySpace space = verify_space(a.ws, a.seqs, pieces, a.tokens_count);
  const int up = t.first + max(t.parent, 0);
  double p = 0.0, q = 0.0, u = 1.0;
  if (t.parent >= 0) {
    const int64_t token = a.tokens[t.first + lane];
    p = prob_at((const float*)a.target + (int64_t)up * a.target_row, token, a.vocab);
    q = prob_at(a.draft + (int64_t)up * a.draft_row, token, a.vocab);
    u = a.accept_u[t.first + lane];
  }
  const bool first_ok = t.parent >= 0 && u * q < positive(p);
  bool eldest = t.parent >= 0, open = true;
  for (uint64_t m = __ballot(t.parent >= 0); m; m &= m - 1) {
    const int e = __builtin_ctzll(m), of = of_lane(t.parent, e), ok = of_lane((int)first_ok, e);
    if (of == t.parent && e < lane) {
      if (eldest) open = !ok;  // e is the first child: only if it was not accepted is this one asked
      eldest = false;
    }
  }
  if (eldest) open = first_ok;
  const uint64_t way = __ballot(t.parent >= 0 && open) | 1;
  const uint64_t mine = of_lane(t.ancestors, node), children = __ballot(t.parent == node);
  int chosen = -1;
  double taken = 0.0, left = 1.0;
  if ((mine & ~way) == 0) {
    const float* const prow = (const float*)a.target + (int64_t)(t.first + node) * a.target_row;
    const float* const qrow = a.draft + (int64_t)(t.first + node) * a.draft_row;
    for (uint64_t m = children; m; m &= m - 1) {
      const int c = __builtin_ctzll(m);
      const double pc = of_lane(p, c), qc = of_lane(q, c), uc = of_lane(u, c);
      if (uc * left * qc < positive(pc - taken * qc)) {
        chosen = c;
        break;
      }
      taken += left;
      if (m & (m - 1)) {
        double sum = 0.0;
        int i = 4 * threadIdx.x;
        for (; i + 4 <= a.vocab; i += 4 * kChooseThreads) {
          const row4_t x = *(const row4_t*)(prow + i), y = *(const row4_t*)(qrow + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += positive(fma(-taken, (double)y[e], (double)x[e]));
        }
        for (; i < a.vocab; ++i) sum += positive(fma(-taken, (double)qrow[i], (double)prow[i]));
        left = block_sum<kChooseThreads>(sum, parts);
      }
    }
  }
  if (threadIdx.x < 64) {
    if (children >> lane & 1) space.chosen[t.first + lane] = lane == chosen;
    if (lane == 0) space.taken[t.first + node] = taken;
  }
}

// Children of each node given as tokens: each accepted with what is left of its parent's mass.
__device__ __forceinline__ bool accept_given(const VerifyArgs& a, const Tree& t, int64_t token, int lane) {
  double p = 0.0, u = 1.0;
  if (t.parent >= 0) {
    p = positive(prob_at((const float*)a.target + (int64_t)(t.first + t.parent) * a.target_row, token, a.vocab));
    u = a.accept_u[t.first + lane];
  }
  double left = 1.0;
  bool again = false;  // an elder has this token
  for (uint64_t m = __ballot(t.parent >= 0); m; m &= m - 1) {
    const int e = __builtin_ctzll(m), of = of_lane(t.parent, e), counted = of_lane((int)again, e);
    const double mass = of_lane(p, e);
    const int64_t other = of_lane(token, e);
    if (of == t.parent && e < lane) {
      again |= other == token;
      left -= counted ? 0.0 : mass;
    }
  }
  return t.parent >= 0 && !again && u * left < p;
}

// A thread's 16 values of a piece: four each of every quarter.
struct PieceValues {
  double f[4][4];
};
template <bool DRAWN>
__device__ __forceinline__ PieceValues piece_values(const float* prow, const float* qrow, double taken, const uint32_t* gone,
                                                    int begin, int vocab) {
  PieceValues v;
  row4_t x[4], y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = 4 * (kPickThreads * j + (int)threadIdx.x), i = begin + at;
    if (i + 4 <= vocab) {
      x[j] = *(const row4_t*)(prow + i);
      if (DRAWN) y[j] = *(const row4_t*)(qrow + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[j][e] = i + e < vocab ? prow[i + e] : 0.0f;
        if (DRAWN) y[j][e] = i + e < vocab ? qrow[i + e] : 0.0f;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = 4 * (kPickThreads * j + (int)threadIdx.x);
    const uint32_t out = DRAWN ? 0 : gone[at >> 5] >> (at & 31);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v.f[j][e] = DRAWN ? positive(fma(-taken, (double)y[j][e], (double)x[j][e])) : out >> e & 1 ? 0.0 : positive(x[j][e]);
  }
  return v;
}
// The bits of a piece's values that are no longer there: the tokens of the last node's children.
__device__ __forceinline__ void mark_gone(uint32_t* gone, bool under, int64_t token, int begin) {
  __syncthreads();
  for (int i = threadIdx.x; i < kPiece / 32; i += kPickThreads) gone[i] = 0;
  __syncthreads();
  if (threadIdx.x < 64 && under && token >= begin && token < begin + kPiece)
    atomicOr(&gone[(token - begin) >> 5], 1u << ((token - begin) & 31));
  __syncthreads();
}

// Workgroup (piece, request).
template <bool DRAWN>
__global__ __launch_bounds__(kPickThreads) void verify_sum_kernel(VerifyArgs a, int pieces) {
  __shared__ double parts[kPickThreads / 64];
  __shared__ uint32_t gone[DRAWN ? 1 : kPiece / 32];
  const int lane = threadIdx.x & 63, piece = blockIdx.x, r = blockIdx.y;
  const VerifySpace space = verify_space(a.ws, a.seqs, pieces, a.tokens_count);
  const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens_count, a.width, lane);
  const int64_t token = lane < t.nodes ? a.tokens[t.first + lane] : -1;
  bool chosen;
  if constexpr (DRAWN) chosen = t.parent >= 0 && space.chosen[t.first + lane];
  else chosen = first_accepted(accept_given(a, t, token, lane), t.parent, lane);
  const uint64_t on = path_of(t, chosen, lane);
  const int last = on ? 63 - __clzll((long long)on) : -1;
  const int row = last < 0 ? -1 : t.first + last;
  const double taken = DRAWN && last >= 0 ? space.taken[row] : 0.0;
  if (piece == 0 && threadIdx.x < 64) {
    write_path(a, r, t, on, token, lane);
    if (lane == 0) space.last[r] = Last{taken, row, last};
  }
  if (last < 0) return;
  if constexpr (!DRAWN) mark_gone(gone, t.parent == last, token, piece * kPiece);
  const PieceValues v = piece_values<DRAWN>((const float*)a.target + (int64_t)row * a.target_row,
                                            DRAWN ? a.draft + (int64_t)row * a.draft_row : nullptr, taken, gone, piece * kPiece,
                                            a.vocab);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += v.f[j][e];
  sum = block_sum<kPickThreads>(sum, parts);
  if (threadIdx.x == 0) space.sums[(int64_t)r * pieces + piece] = sum;
}

// Sums over the threads up to and including each, and of all.
struct Scan {
  double upto, all;
};
__device__ __forceinline__ Scan block_scan(double v, double* parts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double w = __shfl_up(v, off);
    if (lane >= off) v += w;
  }
  __syncthreads();
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) {
    if (w < wave) before += parts[w];
    all += parts[w];
  }
  return Scan{before + v, all};
}

template <bool DRAWN>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs a, int pieces) {
  __shared__ double parts[kPickThreads / 64];
  __shared__ uint32_t gone[DRAWN ? 1 : kPiece / 32];
  __shared__ int found, some;
  __shared__ double found_at;
  const int tid = threadIdx.x, r = blockIdx.x;
  const VerifySpace space = verify_space(a.ws, a.seqs, pieces, a.tokens_count);
  const Last last = space.last[r];
  if (last.row < 0) return;
  const float* const prow = (const float*)a.target + (int64_t)last.row * a.target_row;
  const float* const qrow = DRAWN ? a.draft + (int64_t)last.row * a.draft_row : nullptr;
  const int first = last.row - last.node;
  const int nodes = min(seq_offset(a.cu, r + 1, a.seqs, a.tokens_count) - first, a.width);
  const bool node = tid < nodes;
  const int64_t token = node ? a.tokens[first + tid] : -1;
  bool under = node && tid > last.node && a.parents[first + tid] == last.node;
  double taken = last.a;
  const double* sums = space.sums + (int64_t)r * pieces;

  // What is left may be nothing, where the probabilities do not add up: the token is drawn from all of the row then.
  bool whole = false;
  auto sum_of = [&](int s) { return s < pieces ? sums[s] : 0.0; };
  auto values = [&](int s) {
    if constexpr (!DRAWN) mark_gone(gone, under && !whole, token, s * kPiece);
    return piece_values<DRAWN>(prow, qrow, taken, gone, s * kPiece, a.vocab);
  };
  auto add_up = [&](const PieceValues& v) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += v.f[j][e];
    return block_sum<kPickThreads>(sum, parts);
  };
  double all = 0.0;
  for (int s0 = 0; s0 < pieces; s0 += kPickThreads) all += block_sum<kPickThreads>(sum_of(s0 + tid), parts);
  if (!(all > 0.0)) {
    whole = true;
    taken = 0.0;
    all = 0.0;
    for (int s = 0; s < pieces; ++s) all += add_up(values(s));
  }
  const double mark = (double)a.sample_u[r] * all;

  // The first piece with whose end the sum passes the mark; if none does (a number that is not below 1), the last with any.
  int piece = -1;
  double before = 0.0;
  if (!whole) {
    if (tid == 0) found = 0x7fffffff, some = -1;
    double carry = 0.0;
    for (int s0 = 0; s0 < pieces; s0 += kPickThreads) {
      const double mine = sum_of(s0 + tid);
      const Scan scan = block_scan(mine, parts);  // its barriers are behind the store above
      if (mine > 0.0) {
        atomicMax(&some, s0 + tid);
        if (carry + scan.upto > mark) atomicMin(&found, s0 + tid);
      }
      __syncthreads();
      if (found == s0 + tid) found_at = carry + scan.upto - mine;
      carry += scan.all;
      if (found != 0x7fffffff) break;
    }
    __syncthreads();
    piece = found != 0x7fffffff ? found : some;
    before = found != 0x7fffffff ? found_at : 0.0;
  } else {
    for (int s = 0; s < pieces; ++s) {
      const double sum = add_up(values(s));
      if (sum > 0.0) piece = s;
      if (sum > 0.0 && before + sum > mark) break;
      before += sum;
    }
  }
  __syncthreads();  // both have been read
  if (tid == 0) found = 0x7fffffff, some = piece < 0 ? 0 : -1;
  if (piece >= 0) {
    const PieceValues v = values(piece);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double mine = v.f[j][0] + v.f[j][1] + v.f[j][2] + v.f[j][3];
      const Scan scan = block_scan(mine, parts);
      double upto = before + (scan.upto - mine);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        upto += v.f[j][e];
        const int i = piece * kPiece + 4 * (kPickThreads * j + tid) + e;
        if (v.f[j][e] > 0.0) {
          atomicMax(&some, i);
          if (upto > mark) atomicMin(&found, i);
        }
      }
      before += scan.all;
    }
  }
  __syncthreads();
  if (tid == 0) a.emitted[(int64_t)r * a.width + a.counts[r] - 1] = found != 0x7fffffff ? found : some;
}

// ---- what is kept -----------------------------------------------------------------------------------------------
// Node path[i] of the tree goes to place context + i, in all arrays of the cache.  Nodes have larger numbers than their
// ancestors, so path[i] >= i, and a place is read before it is written if every thread takes the moves of its 16 bytes in
// order.  Bound by latency: the offsets of the moves by way of the table, then a read and a write.  Workgroup (r, y): share y of
// the arrays of request r; r = seqs: the lengths, and the pages behind them back onto the stack.
constexpr int kKeepThreads = 256, kKeepAhead = 4;

__device__ __forceinline__ int kept_tokens(const KeepArgs& a, int r) {
  const int context = max(load_const(a.context_lens, r), 0), seq = max(load_const(a.seq_lens, r), context);
  return context + min(min(max(load_const(a.counts, r), 0), a.width), seq - context);
}

__global__ __launch_bounds__(kKeepThreads) void keep_drafts_kernel(KeepArgs a) {
  __shared__ int64_t src[kNodes], dst[kNodes];
  __shared__ int moves, scan[kKeepThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, r = blockIdx.x;
  const int block = (1 << a.log2_block) - 1;
  if (r == a.seqs) {
    if (blockIdx.y) return;
    // Every thread takes a run of requests: what they give back is counted, then written behind what the ones before give.
    const int64_t cap = (int64_t)a.table_width << a.log2_block;
    const int run = (a.seqs + kKeepThreads - 1) / kKeepThreads, r0 = min(tid * run, a.seqs), r1 = min(r0 + run, a.seqs);
    const bool pages = a.free_count != nullptr;
    const int count = pages ? min(max(load_const(a.free_count, 0), 0), a.free_capacity) : 0;
    auto spare = [&](int s, auto&& take) {
      if (!pages) return;
      const int64_t kept = kept_tokens(a, s), held = max(load_const(a.seq_lens, s), 0);
      const int need = (int)((min(kept, cap) + block) >> a.log2_block);
      for (int p = need; p < (int)((min(held, cap) + block) >> a.log2_block); ++p) {
        const int page = a.table[(int64_t)s * a.table_stride + p];
        if (page >= 0) take(page);
      }
    };
    int mine = 0;
    for (int s = r0; s < r1; ++s) spare(s, [&](int) { ++mine; });
    const int upto = wave_prefix(mine);
    if (lane == 63) scan[tid >> 6] = upto;
    __syncthreads();
    int64_t at = count + (int64_t)upto - mine, all = count;
#pragma unroll
    for (int w = 0; w < kKeepThreads / 64; ++w) {
      if (w < tid >> 6) at += scan[w];
      all += scan[w];
    }
    for (int s = r0; s < r1; ++s) {
      spare(s, [&](int page) {
        if (at < a.free_capacity) a.free_pages[at] = page;
        ++at;
      });
      if (a.kept_lens) a.kept_lens[s] = kept_tokens(a, s);
    }
    if (pages && tid == 0) *a.free_left = (int)min(all, (int64_t)a.free_capacity);
    return;
  }

  if (tid < 64) {
    const int context = max(load_const(a.context_lens, r), 0), count = kept_tokens(a, r) - context;
    const int from = lane < count ? a.path[(int64_t)r * a.path_stride + lane] : lane;
    auto offset = [&](int64_t token) {  // of a token's entry in its page's array; -1: not in the cache
      const int64_t p = token >> a.log2_block;
      const int page = p < a.table_width ? a.table[(int64_t)r * a.table_stride + p] : -1;
      return (unsigned)page < (unsigned)a.num_pages ? page * a.page_stride + (token & block) * a.token_stride : (int64_t)-1;
    };
    int64_t s = -1, d = -1;
    if (from > lane && from < kNodes) {
      s = offset((int64_t)context + from);
      d = offset((int64_t)context + lane);
    }
    const uint64_t move = __ballot(s >= 0 && d >= 0);
    if (move >> lane & 1) {
      const int i = __popcll(move & ((1ull << lane) - 1));
      src[i] = s;
      dst[i] = d;
    }
    if (lane == 0) moves = __popcll(move);
  }
  __syncthreads();
  const int n = moves;
  if (n == 0) return;
  const int pieces = a.head_dim / 8, per_array = a.kv_heads * pieces;
  const int64_t all = (int64_t)a.arrays * per_array;
  for (int64_t i = (int64_t)blockIdx.y * kKeepThreads + tid; i < all; i += (int64_t)gridDim.y * kKeepThreads) {
    const int64_t array = i / per_array;
    const int c = (int)(i - array * per_array), head = c / pieces;
    uint16_t* const base = (uint16_t*)a.caches + array * a.array_stride + head * a.head_stride + 8 * (c - head * pieces);
    for (int m = 0; m < n; m += kKeepAhead) {
      u32x4 x[kKeepAhead];
#pragma unroll
      for (int j = 0; j < kKeepAhead; ++j)
        if (m + j < n) x[j] = *(const u32x4*)(base + src[m + j]);
#pragma unroll
      for (int j = 0; j < kKeepAhead; ++j)
        if (m + j < n) *(u32x4*)(base + dst[m + j]) = x[j];
    }
  }
}

int row_pieces(int vocab) { return (int)(((int64_t)vocab + kPiece - 1) / kPiece); }

// Workgroups per row of scores, where there are fewer rows than fill the card, of at least four rounds of loads.
int row_shares(const VerifyArgs& a) {
  const int64_t most = ((int64_t)a.vocab + 4 * kBestStep - 1) / (4 * kBestStep);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, 1024 / std::max(a.tokens_count, 1)));
}

template <class T>
void best_launch(const VerifyArgs& a, int shares, hipStream_t stream) {
  const int part = (int)((((int64_t)a.vocab + shares - 1) / shares + kBestStep - 1) / kBestStep * kBestStep);
  best_token_kernel<T><<<a.tokens_count * shares, kBestThreads, 0, stream>>>(a, shares, part);
}

template <bool DRAWN>
hipError_t sample_launch(const VerifyArgs& a, hipStream_t stream) {
  const int pieces = row_pieces(a.vocab);
  if (DRAWN) choose_child_kernel<<<dim3(a.width, a.seqs), kChooseThreads, 0, stream>>>(a, pieces);
  verify_sum_kernel<DRAWN><<<dim3(pieces, a.seqs), kPickThreads, 0, stream>>>(a, pieces);
  verify_pick_kernel<DRAWN><<<a.seqs, kPickThreads, 0, stream>>>(a, pieces);
  return hipGetLastError();
}

}  // namespace

hipError_t draft_trees_launch(const DraftTreesArgs& a, hipStream_t stream) {
  draft_trees_kernel<<<(a.seqs + kTreeWaves - 1) / kTreeWaves, 64 * kTreeWaves, 0, stream>>>(a);
  return hipGetLastError();
}

size_t verify_workspace_bytes(const VerifyArgs& a) {
  if (a.mode == kVerifyBest) return (size_t)a.tokens_count * row_shares(a) * sizeof(uint64_t);
  const VerifySpace s = verify_space(nullptr, a.seqs, row_pieces(a.vocab), a.tokens_count);
  return a.mode == kVerifyDrawn ? (size_t)(s.chosen + a.tokens_count) : (size_t)s.taken;
}

hipError_t verify_launch(const VerifyArgs& a, int dtype, hipStream_t stream) {
  if (a.mode != kVerifyBest) return a.mode == kVerifyDrawn ? sample_launch<true>(a, stream) : sample_launch<false>(a, stream);
  const int shares = row_shares(a);
  if (a.tokens_count > 0) {
    if (dtype == kQuantF32) best_launch<float>(a, shares, stream);
    else if (dtype == kQuantF16) best_launch<half_t>(a, shares, stream);
    else best_launch<bhalf_t>(a, shares, stream);
    if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  }
  verify_best_kernel<<<(a.seqs + kTreeWaves - 1) / kTreeWaves, 64 * kTreeWaves, 0, stream>>>(a, shares);
  return hipGetLastError();
}

hipError_t keep_drafts_launch(const KeepArgs& a, hipStream_t stream) {
  const int64_t pieces = (int64_t)a.arrays * a.kv_heads * (a.head_dim / 8);
  const int64_t shares = std::min<int64_t>((pieces + kKeepThreads - 1) / kKeepThreads, std::max(1, 4096 / (a.seqs + 1)));
  keep_drafts_kernel<<<dim3(a.seqs + 1, (unsigned)std::max<int64_t>(shares, 1)), kKeepThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace kf
