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
};
__device__ __forceinline__ Tree load_tree(const int* parents, const int* cu, int r, int seqs, int tokens, int most, int lane) {
  Tree t;
  t.first = seq_offset(cu, r, seqs, tokens);
  t.len = max(seq_offset(cu, r + 1, seqs, tokens) - t.first, 0);
  t.nodes = min(t.len, most);
  const int p = lane < t.nodes ? parents[t.first + lane] : -1;
  t.parent = (unsigned)p < (unsigned)lane ? p : -1;
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
// A wavefront per request.  Bound by latency: the offsets, then the parents, then six rounds of lane exchange: 1.6 us for one
// tree of 16 nodes, 2.7 for 500 of up to 64.
constexpr int kTreeWaves = 4;

__global__ __launch_bounds__(64 * kTreeWaves) void draft_trees_kernel(DraftTreesArgs a) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * kTreeWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r < a.seqs) {
    const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens, kNodes, lane);
    const int64_t context = (int64_t)load_const(a.seq_lens, r) - t.len;
    // Pointers doubled: after n rounds a node knows 2^n - 1 ancestors and where the next one is.  A root points to itself.
    uint64_t ancestors = 1ull << lane;
    int jump = t.parent < 0 ? lane : t.parent;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      ancestors |= __shfl(ancestors, jump);
      jump = __shfl(jump, jump);
    }
    for (int i = lane; i < t.len; i += 64) {  // past the 64th: no node
      a.ancestors[t.first + i] = i < kNodes ? ancestors : 0;
      a.positions[t.first + i] = i < kNodes ? context + __popcll(ancestors) - 1 : -1;
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
// Whether a child is accepted depends on itself and its elder siblings only, so every lane judges its own node first; then the path
// is one ballot a step.

// From node 0 (which is given) along the first accepted children: the path's nodes.
__device__ __forceinline__ uint64_t path_of(const Tree& t, bool accepted) {
  if (t.nodes == 0) return 0;
  uint64_t on = 1;
  int at = 0;
  while (const uint64_t next = __ballot(accepted && t.parent == at)) {
    at = __builtin_ctzll(next);
    on |= 1ull << at;
  }
  return on;
}
__device__ __forceinline__ int last_of(uint64_t on) { return on ? 63 - __clzll((long long)on) : -1; }

// counts, path and emitted tokens of request r but for the token behind the path; last: the path's last node.
__device__ __forceinline__ void write_path(const VerifyArgs& a, int r, uint64_t on, int64_t token, int lane) {
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

constexpr int kBestThreads = 256, kBestAhead = 4, kBestStep = 8 * kBestThreads;

// keys[row * shares + share] = the largest of the share's part of the row.  Bound by memory: a thread keeps the largest value
// and the eight that it is among, which it reads again at the end, so that a value costs two vector instructions in place of
// five.  464 rows of 100003 bf16 values, 93 MB, take 17.7 us, 5.2 TB/s (with a key for every value 30); 16 of 32000 3.8.
template <class T>
__global__ __launch_bounds__(kBestThreads) void best_token_kernel(VerifyArgs a, int shares, int part) {
  __shared__ uint64_t keys[kBestThreads / 64];
  const int row = blockIdx.x / shares, share = blockIdx.x - row * shares;
  if (row >= seq_offset(a.cu, a.seqs, a.seqs, a.tokens_count)) return;
  const T* const src = (const T*)a.target + (int64_t)row * a.target_row;
  const int begin = share * part, end = min(begin + part, a.vocab), tid = threadIdx.x;
  // A row of 16-bit values may begin between two words: its first value is taken alone.
  const int odd = sizeof(T) == 2 ? (int)((uintptr_t)(src + begin) >> 1 & 1) : 0;
  float best = -__builtin_inff();
  int group = -1;  // of eight values from begin + odd + 8 group on; -1: none above -inf
  const int groups = (end - begin - odd) / 8;
  auto above = [](float x, float y) { return !(x <= y) && y == y; };  // NaN above all numbers
  auto look = [&](const float(&x)[8], int g) {
    const float m0 = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[0], x[1]), x[2]);
    const float m1 = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[3], x[4]), x[5]);
    const float m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_elementwise_maximum(x[6], x[7]), m0), m1);
    if (above(m, best)) {
      best = m;
      group = g;
    }
  };
  int g = tid;
  for (; g + (kBestAhead - 1) * kBestThreads < groups; g += kBestAhead * kBestThreads) {
    float x[kBestAhead][8];
#pragma unroll
    for (int n = 0; n < kBestAhead; ++n) load8(src + begin + odd + 8 * (g + n * kBestThreads), x[n]);
#pragma unroll
    for (int n = 0; n < kBestAhead; ++n) look(x[n], g + n * kBestThreads);
  }
  for (; g < groups; g += kBestThreads) {
    float x[8];
    load8(src + begin + odd + 8 * g, x);
    look(x, g);
  }
  uint64_t key = 0;
  auto offer = [&](float x, int i) {
    const uint64_t k = score_key(x, i);
    key = k > key ? k : key;
  };
  if (group >= 0)
    for (int e = 0; e < 8; ++e) offer((float)src[begin + odd + 8 * group + e], begin + odd + 8 * group + e);
  // The values before and behind the groups, and the first of all, in case they are all -inf.
  const int rest = begin + odd + 8 * groups;
  if (tid < 8 && rest + tid < end) offer((float)src[rest + tid], rest + tid);
  if (tid == 0 && begin < end) offer((float)src[begin], begin);
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

// A wavefront per request.  Latency, 2.3 us for one, 3.9 for 16: the tree, a node's keys, a round of exchange for every node of the
// path.
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
  const uint64_t on = path_of(t, accepted);
  write_path(a, r, on, token, lane);
  if (lane == last_of(on)) a.emitted[(int64_t)r * a.width + __popcll(on) - 1] = best;
}

// ---- from probabilities and given random numbers -------------------------------------------------------------
// What is left of row t's mass after its rejected children is f = max(p - a q, 0) where they were drawn from q, f = p without their
// tokens where they were given.  The token behind the path is the one at which the running sum of f passes u times all of it: a
// sum over the row, then the place in it.  In 64 bits, as an index is an integer and 32 bits would move it.
//
// A workgroup per request does this, the sum in 16 parts, one a wavefront, then the part, or the part of the part, that the place
// is in.  Long rows are first added up by a launch of their own, in pieces of 4096 values: which row it is, is known from the first
// test of every node's first child, unless a later child is accepted.
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64, kPiece = 4 * kPickThreads;
constexpr int kSubs = 4;  // pieces of a 16th whose sums are kept: rows of up to 2^18 values are searched at once
constexpr int kSumThreads = 256;

// Nothing for negative values and NaN.
__device__ __forceinline__ double positive(double x) { return __builtin_fmax(x, 0.0); }
__device__ __forceinline__ float positive(float x) { return __builtin_fmaxf(x, 0.0f); }

// A draft's probability: from 0, which is also NaN's, to 1.  Infinity or NaN times an `a` of 0 (a node without children) would be
// none, and the target's mass there lost.  Costs nothing: the conversion to 64 bits clamps.
__device__ __forceinline__ double drawn_from(float q) { return __builtin_fmin(__builtin_fmax((double)q, 0.0), 1.0); }

// Sums over a wavefront's lanes up to and including each.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_dpp(double v) {
  const u32x2 w = bit_cast<u32x2>(v);
  const u32x2 x = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[0], CTRL, ROWS, 0xF, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[1], CTRL, ROWS, 0xF, false)};
  return v + bit_cast<double>(x);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = add_dpp<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v = add_dpp<0x112, 0xF>(v);
  v = add_dpp<0x114, 0xF>(v);
  v = add_dpp<0x118, 0xF>(v);
  v = add_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return add_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ double wave_sum(double v) { return of_lane(wave_scan(v), 63); }

// A request's tree in LDS: the walk along it is one wavefront's, all others go by what it leaves here.
struct WalkShared {
  uint64_t children[kNodes];
  int64_t token[kNodes];
  double p[kNodes], q[kNodes], u[kNodes];  // of a node's token in its parent's rows, and its random number
  int again[kNodes];                       // an elder sibling has the same token
  int64_t gone[kNodes];                    // the tokens of the path's last node's children
  uint64_t on, under;
  int first, last;
  double taken;
};

// The path as far as it is known without a sum, and the row of its last node with what is taken off.
struct Way {
  uint64_t on;
  int first, last;  // last -1: the request has no nodes
  uint64_t under;   // the last node's children
  double taken;
};

// By one wavefront: the tests that need no sum, and the path that they make.  Children given as tokens: each is accepted with what
// is left of its parent's mass, of several with one token the first.  Children that were drawn: the first of each node.
template <bool DRAWN>
__device__ __forceinline__ void walk(const VerifyArgs& a, WalkShared& sh, int r, int lane) {
  const Tree t = load_tree(a.parents, a.cu, r, a.seqs, a.tokens_count, a.width, lane);
  sh.children[lane] = 0;
  if (t.nodes > 0) {  // the same for all lanes
    const int mine = t.first + min(lane, t.nodes - 1), up = t.first + max(t.parent, 0);
    const int64_t token = a.tokens[mine], inside = token >= 0 && token < a.vocab ? token : 0;
    const float u = a.accept_u[mine], p = ((const float*)a.target)[(int64_t)up * a.target_row + inside];
    const double q = DRAWN ? drawn_from(a.draft[(int64_t)up * a.draft_row + inside]) : 0.0;
    const bool real = token == inside;  // others have no mass
    sh.token[lane] = token;
    sh.p[lane] = real ? positive(p) : 0.0;
    sh.q[lane] = real ? q : 0.0;
    sh.u[lane] = u;
    if (t.parent >= 0)
      atomicOr((unsigned long long*)&sh.children[t.parent], 1ull << lane);  // by one wavefront, an or: no order to it
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const uint64_t elders = t.parent >= 0 ? sh.children[t.parent] & ((1ull << lane) - 1) : 0;
  bool accepted = false;
  if constexpr (DRAWN) {
    accepted = t.parent >= 0 && elders == 0 && sh.u[lane] * sh.q[lane] < sh.p[lane];
  } else {
    bool again = false;
    if (t.parent >= 0)
      for (uint64_t m = elders; m; m &= m - 1) again |= sh.token[__builtin_ctzll(m)] == sh.token[lane];
    sh.again[lane] = again;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (t.parent >= 0) {
      double left = 1.0;
      for (uint64_t m = elders; m; m &= m - 1) {
        const int e = __builtin_ctzll(m);
        left -= sh.again[e] ? 0.0 : sh.p[e];
      }
      accepted = !again && sh.p[lane] > 0.0 && sh.u[lane] * left < sh.p[lane];  // `left` may be negative, and numbers too
    }
  }
  const uint64_t on = path_of(t, accepted);
  const int last = last_of(on);
  const uint64_t under = __ballot(t.parent == last && last >= 0);
  if (under >> lane & 1) sh.gone[__popcll(under & ((1ull << lane) - 1))] = sh.token[lane];
  if (lane == 0) {
    sh.on = on;
    sh.under = under;
    sh.first = t.first;
    sh.last = last;
    sh.taken = DRAWN && under ? 1.0 : 0.0;
  }
}
// Of all wavefronts, behind a barrier: the same in all lanes, and known to be.
__device__ __forceinline__ Way way_of(const WalkShared& sh) {
  Way w;
  w.on = of_lane(sh.on, 0);
  w.under = of_lane(sh.under, 0);
  w.first = of_lane(sh.first, 0);
  w.last = of_lane(sh.last, 0);
  w.taken = of_lane(sh.taken, 0);
  return w;
}

// Values of f in a row.
template <bool DRAWN>
struct Rest {
  const float* p;
  const float* q;
  const int64_t* gone;  // LDS: tokens that are out of it
  int gone_count, vocab;
  double taken;

  // Four values from i on; `from` and the next 4 x LANES values are what the lanes that come here together look at.
  template <int LANES>
  __device__ __forceinline__ void four(row4_t x, row4_t y, int i, int from, double (&f)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = DRAWN ? positive(fma(-taken, drawn_from(y[e]), (double)x[e])) : (double)positive(x[e]);
    if constexpr (!DRAWN) {
      for (int g = 0; g < gone_count; ++g) {
        const int64_t token = gone[g];
        if (token >= from && token < from + 4 * LANES) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e == token) f[e] = 0.0;
        }
      }
    }
  }
  __device__ __forceinline__ row4_t load(const float* row, int i, int end) const {  // zeros from `end` on
    if (i + 4 <= end) return *(const row4_t*)(row + i);
    row4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < end ? row[i + e] : 0.0f;
    return v;
  }
  // The sum over [begin, end) by one wavefront, the same in all lanes: in groups of four values, of which the next come while
  // the present ones are added up, then up to three values alone.  KEEP: subs has those of each 4096 values, the first kSubs.
  template <bool KEEP>
  __device__ __forceinline__ double wave_total(int begin, int end, int lane, double* subs) const {
    constexpr int AHEAD = 4;
    static_assert(kPiece % (4 * 64 * AHEAD) == 0, "a piece ends with a round of loads");
    double all = 0.0, sum = 0.0;
    const int groups = max(end - begin, 0) / 4;
    auto next_piece = [&](int at) {  // of the values from `begin` on
      if (!KEEP || at == 0 || at % kPiece != 0) return;
      const double one = wave_sum(sum);
      if (lane == 0 && at <= kSubs * kPiece) subs[at / kPiece - 1] = one;
      all += one;
      sum = 0.0;
    };
    if (groups > 0) {
      row4_t x[AHEAD], y[AHEAD];
      auto load_group = [&](int j, int g) {
        const int i = begin + 4 * (g < groups ? g : 0);  // past the last one: the first, for nothing
        x[j] = *(const row4_t*)(p + i);
        if (DRAWN) y[j] = *(const row4_t*)(q + i);
      };
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) load_group(j, 64 * j + lane);
      for (int g0 = 0; g0 < groups; g0 += 64 * AHEAD) {
        next_piece(4 * g0);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int g = g0 + 64 * j + lane;
          double f[4];
          four<64>(x[j], y[j], begin + 4 * g, begin + 4 * (g0 + 64 * j), f);
          const double four_of = (f[0] + f[1]) + (f[2] + f[3]);
          sum += g < groups ? four_of : 0.0;
          load_group(j, g + 64 * AHEAD);
        }
      }
    }
    next_piece(4 * groups);
    const int rest = begin + 4 * groups;
    if (rest + lane < end) {
      double f[4];
      four<64>(row4_t{p[rest + lane], 0.0f, 0.0f, 0.0f}, row4_t{DRAWN ? q[rest + lane] : 0.0f, 0.0f, 0.0f, 0.0f},
               rest + lane, rest, f);
      sum += f[0];
    }
    const double one = wave_sum(sum);
    if (KEEP && lane == 0)
      for (int i = 4 * groups / kPiece, first = i; i < kSubs; ++i) subs[i] = i == first ? one : 0.0;
    return all + one;
  }
};
template <bool DRAWN>
__device__ __forceinline__ Rest<DRAWN> rest_of(const VerifyArgs& a, const WalkShared& sh, const Way& w) {
  const int64_t row = w.first + w.last;
  return Rest<DRAWN>{(const float*)a.target + row * a.target_row, DRAWN ? a.draft + row * a.draft_row : nullptr, sh.gone,
                     DRAWN ? 0 : (int)__popcll(w.under), a.vocab, w.taken};
}

// The workspace where rows are summed by a launch of their own; again and come: DRAWN.
struct PickSpace {
  double* sums;    // [seqs][pieces]
  double* again;   // the same with more taken off
  uint32_t* come;  // [seqs] workgroups whose pieces are in `again`
};
__device__ __host__ __forceinline__ PickSpace pick_space(const VerifyArgs& a, int pieces) {
  double* const sums = static_cast<double*>(a.ws);
  double* const again = sums + (int64_t)a.seqs * pieces;
  return PickSpace{sums, again, reinterpret_cast<uint32_t*>(again + (int64_t)a.seqs * pieces)};
}

// Workgroup (piece, request): the sum over the piece.  16 rows of 150001 values of p and of q, 19 MB, take 6.3 us, the walk before
// them included.
template <bool DRAWN>
__global__ __launch_bounds__(kSumThreads) void verify_sum_kernel(VerifyArgs a, int pieces) {
  __shared__ double parts[kSumThreads / 64];
  __shared__ WalkShared walked;
  const int lane = threadIdx.x & 63, piece = blockIdx.x, r = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (DRAWN && piece == 0 && threadIdx.x == 0) pick_space(a, pieces).come[r] = 0;
  if (wave == 0) walk<DRAWN>(a, walked, r, lane);
  __syncthreads();
  const Way w = way_of(walked);
  if (w.last < 0) return;
  const Rest<DRAWN> rest = rest_of<DRAWN>(a, walked, w);
  constexpr int MINE = kPiece / (kSumThreads / 64);
  const int begin = piece * kPiece + wave * MINE;
  const double sum = rest.template wave_total<false>(begin, min(begin + MINE, a.vocab), lane, nullptr);
  if (lane == 0) parts[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    pick_space(a, pieces).sums[(int64_t)r * pieces + piece] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

struct PickShared {
  WalkShared walked;
  double parts[kPickWaves], subs[kPickWaves][kSubs], scan[kPickWaves];
  double before;
  int low[kPickWaves], high[kPickWaves];
  int goes_on;
};

// Sums over the threads up to and including each, and of all.
struct Scan {
  double upto, all;
};
__device__ __forceinline__ Scan block_scan(double v, PickShared& sh, int lane, int wave) {
  v = wave_scan(v);
  __syncthreads();  // the last scan's have been read
  if (lane == 63) sh.scan[wave] = v;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) {
    if (w < wave) before += sh.scan[w];
    all += sh.scan[w];
  }
  return Scan{before + v, all};
}

// The lowest and the highest number that any thread has (0x7fffffff and -1: none), where numbers ascend with the threads.
struct Ends {
  int low, high;
};
__device__ __forceinline__ Ends ends_of(int low, int high, PickShared& sh, int lane, int wave) {
  const uint64_t lows = __ballot(low != 0x7fffffff), highs = __ballot(high >= 0);
  const int l = lows ? of_lane(low, __builtin_ctzll(lows)) : 0x7fffffff;
  const int h = highs ? of_lane(high, 63 - __clzll((long long)highs)) : -1;
  __syncthreads();
  if (lane == 0) {
    sh.low[wave] = l;
    sh.high[wave] = h;
  }
  __syncthreads();
  Ends e = {0x7fffffff, -1};
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) {
    e.low = min(e.low, sh.low[w]);
    e.high = max(e.high, sh.high[w]);
  }
  return e;
}

// The same where they do not: rows of more than 2^22 values.
__device__ __forceinline__ Ends lowest_of(int low, int high, PickShared& sh, int lane, int wave) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    low = min(low, __shfl_xor(low, off));
    high = max(high, __shfl_xor(high, off));
  }
  return ends_of(lane == 0 ? low : 0x7fffffff, lane == 0 ? high : -1, sh, lane, wave);
}

// The sum over the row, a 16th of it by each wavefront; those stay in sh.parts, and (DRAWN: others add up short rows only) their
// pieces' in sh.subs.
template <bool DRAWN>
__device__ __forceinline__ double row_total(PickShared& sh, const Rest<DRAWN>& rest, int begin, int end, int lane, int wave) {
  const int part = ((end - begin + kPickWaves - 1) / kPickWaves + 3) & ~3;
  const int64_t at = begin + (int64_t)part * wave;
  const double mine =
      rest.template wave_total<DRAWN>((int)min(at, (int64_t)end), (int)min(at + part, (int64_t)end), lane, sh.subs[wave]);
  __syncthreads();
  if (lane == 0) sh.parts[wave] = mine;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) all += sh.parts[w];
  return all;
}

// By all workgroups of a request: the sums over the pieces once more, to `again`.  True in the one that is last done.
template <bool DRAWN>
__device__ __forceinline__ bool add_together(const VerifyArgs& a, PickShared& sh, const Rest<DRAWN>& rest, double* again,
                                             int pieces, int lane, int wave) {
  for (int p0 = 4 * blockIdx.y; p0 < pieces; p0 += 4 * gridDim.y) {
    const int piece = p0 + wave / 4, begin = piece * kPiece + wave % 4 * (kPiece / 4);
    const double sum = rest.template wave_total<false>(min(begin, a.vocab), min(begin + kPiece / 4, a.vocab), lane, nullptr);
    __syncthreads();
    if (lane == 0) sh.parts[wave] = sum;
    __syncthreads();
    const double* const four = sh.parts + wave;  // as verify_sum_kernel adds them
    if (lane == 0 && wave % 4 == 0 && piece < pieces)
      __hip_atomic_store(again + piece, (four[0] + four[1]) + (four[2] + four[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // The sums are atomics of the whole device's scope, which go past the caches that XCDs have of their own: there once they are
  // acknowledged, before the barrier, and so before the count.  (Fences of that scope write back and empty the caches: 10 us.)
  // The language would have those fences: without them this holds for the processors named here, whose stores are counted with
  // the loads (vmcnt) and acknowledged where the whole device sees them.
#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "add_together: sums are handed on as gfx950 orders them; other processors need a release and an acquire here"
#endif
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    sh.goes_on = __hip_atomic_fetch_add(pick_space(a, pieces).come + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 gridDim.y - 1;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(sh.goes_on) != 0;
}

// One workgroup per request, or (DRAWN) several of which one goes on.  pieces: of the rows, whose sums the launch before has
// left in a.ws; 0: there was none.  64 requests over 32000 values, tokens given, 12.1 us (with an LDS atomic for every value
// that may be the place 60).  Drawn, bound by what CUs read: each child that is tested behind a node's first costs a sum over the
// row that is left then, 1.2 MB of 150001 values, 11 us by one CU (10.5 with 32-bit products), 3 by ten.  Both launches of 16 such
// requests: 12.5 us without such children, 15.7 with one, 28 with two (one workgroup each 26 and 37.5; a launch of all CUs for
// these sums 30 for two, but 15.5 for none).
template <bool DRAWN>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs a, int pieces) {
  __shared__ PickShared sh;
  WalkShared& walked = sh.walked;
  const int tid = threadIdx.x, lane = tid & 63, r = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const double* sums = pick_space(a, pieces).sums + (int64_t)r * pieces;
  const float sample_u = a.sample_u[r];
  double my_sum = tid < pieces ? sums[tid] : 0.0;
  if (wave == 0) walk<DRAWN>(a, walked, r, lane);
  __syncthreads();
  Way w = way_of(walked);
  if (w.last < 0) {
    if (wave == 0 && blockIdx.y == 0) write_path(a, r, 0, 0, lane);
    return;
  }
  bool summed = pieces > 0;  // the pieces' sums are those of the present row and what is taken off
  auto add_pieces = [&] {
    double sum = my_sum;
    for (int i = tid + kPickThreads; i < pieces; i += kPickThreads) sum += sums[i];
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) sh.parts[wave] = sum;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int v = 0; v < kPickWaves; ++v) all += sh.parts[v];
    return all;
  };
  // Drawn: the last node's further children, each of whose tests needs the sum of what the ones before have left; the first one has
  // been rejected.  Then the sum of what is left to draw from.
  uint64_t open = DRAWN ? w.under & (w.under - 1) : 0;
  auto test = [&](double all) {  // of the first open child
    const int c = __builtin_ctzll(open);
    open &= open - 1;
    if (!(walked.u[c] * all * walked.q[c] < positive(walked.p[c] - w.taken * walked.q[c]))) {
      w.taken += all;
      return;
    }
    // Accepted: on along first children, as far as they are.
    w.on |= 1ull << c;
    w.last = c;
    while (true) {
      w.under = of_lane(walked.children[w.last], 0);
      w.taken = w.under ? 1.0 : 0.0;
      open = w.under & (w.under - 1);
      if (!w.under) break;
      const int e = __builtin_ctzll(w.under);
      if (!(walked.u[e] * walked.q[e] < walked.p[e])) break;
      w.on |= 1ull << e;
      w.last = e;
    }
  };
  // The workgroups of a request make the first of these tests all together.  If there is none, the first one goes on alone.  If
  // there is, each adds up some of the pieces of what is left then, and the one that is last done goes on: none waits for another.
  if (DRAWN && gridDim.y > 1) {  // a thread has all of the sums that it reads: pick_team
    bool on = blockIdx.y == 0;
    if (open) {
      test(add_pieces());
      sums += (int64_t)a.seqs * pieces;
      on = add_together<DRAWN>(a, sh, rest_of<DRAWN>(a, walked, w), const_cast<double*>(sums), pieces, lane, wave);
      if (on) my_sum = tid < pieces ? __hip_atomic_load(sums + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    }
    if (!on) return;
  }
  bool whole = false;
  double all;
  Rest<DRAWN> rest;
  while (true) {
    rest = rest_of<DRAWN>(a, walked, w);
    if (whole) {
      rest.taken = 0.0;
      rest.gone_count = 0;
    }
    all = summed ? add_pieces() : row_total(sh, rest, 0, a.vocab, lane, wave);
    if (open) {
      test(all);
      summed = false;
    } else if (all > 0.0 || whole) {
      break;
    } else {
      whole = true;  // nothing is left, where the probabilities do not add up: the token is drawn from all of the row
      summed = false;
    }
  }
  if (wave == 0) write_path(a, r, w.on, walked.token[lane], lane);
  const double mark = (double)sample_u * all;

  // The part of [begin, end) with whose end the sum passes the mark; if none does (a number that is not below 1), the last
  // with any.
  double before = 0.0;
  int begin = 0, end = a.vocab;
  if (summed) {
    double carry = 0.0, low_at = 0.0;
    int low = 0x7fffffff, high = -1;
    for (int i0 = 0; i0 < pieces; i0 += kPickThreads) {
      const double mine = i0 == 0 ? my_sum : i0 + tid < pieces ? sums[i0 + tid] : 0.0;
      const Scan scan = block_scan(mine, sh, lane, wave);
      if (mine > 0.0) {
        high = i0 + tid;
        if (low == 0x7fffffff && carry + scan.upto > mark) low = i0 + tid, low_at = carry + (scan.upto - mine);
      }
      carry += scan.all;
    }
    const Ends e = pieces <= kPickThreads ? ends_of(low, high, sh, lane, wave) : lowest_of(low, high, sh, lane, wave);
    if (low == e.low && low != 0x7fffffff) sh.before = low_at;
    __syncthreads();
    const int piece = e.low != 0x7fffffff ? e.low : max(e.high, 0);
    before = e.low != 0x7fffffff ? sh.before : 0.0;
    begin = piece * kPiece;
    end = min(begin + kPiece, a.vocab);
  }
  // The one of some sums.
  auto find = [&](const double* parts, int count) {
    int at = -1, some = 0;
    double upto = before, found = 0.0;
    for (int v = 0; v < count; ++v) {
      const double sum = parts[v];
      if (sum > 0.0) some = v;
      if (at < 0 && sum > 0.0 && upto + sum > mark) at = v, found = upto;
      upto += sum;
    }
    before = found;
    return at >= 0 ? at : some;
  };
  while (end - begin > kPiece) {
    if (begin != 0 || end != a.vocab) row_total(sh, rest, begin, end, lane, wave);  // the whole row's parts are there
    const int part = ((end - begin + kPickWaves - 1) / kPickWaves + 3) & ~3, at = find(sh.parts, kPickWaves);
    begin = min(begin + at * part, end);
    end = min(begin + part, end);
    if (DRAWN && part > kPiece && part <= kSubs * kPiece) {
      begin = min(begin + find(sh.subs[at], kSubs) * kPiece, end);
      end = min(begin + kPiece, end);
    }
    __syncthreads();  // the parts have been read
  }
  const int i = begin + 4 * tid;
  double f[4];
  rest.template four<kPickThreads>(rest.load(rest.p, i, end), DRAWN ? rest.load(rest.q, i, end) : row4_t{}, i, begin, f);
  const double mine = (f[0] + f[1]) + (f[2] + f[3]);
  const Scan scan = block_scan(mine, sh, lane, wave);
  double upto = before + (scan.upto - mine);
  int low = 0x7fffffff, high = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    upto += f[e];
    if (f[e] > 0.0) {
      high = i + e;
      if (low == 0x7fffffff && upto > mark) low = i + e;
    }
  }
  const Ends e = ends_of(low, high, sh, lane, wave);
  if (tid == 0) a.emitted[(int64_t)r * a.width + __popcll(w.on) - 1] = e.low != 0x7fffffff ? e.low : max(e.high, 0);
}

// ---- what is kept -----------------------------------------------------------------------------------------------
// Node path[i] of the tree goes to place context + i, in all arrays of the cache.  Nodes have larger numbers than their
// ancestors, so path[i] >= i, and a place is read before it is written if every thread takes the moves of its 16 bytes in
// order.  Bound by latency: the offsets of the moves by way of the table, then a read and a write.  Workgroup (r, y): share y of
// the arrays of request r; r = seqs: the lengths, and the pages behind them back onto the stack.  3.3 us for one request in 44
// arrays, 3.7 for 64 in 56 (3 MB).
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

// Rows up to which one workgroup adds them up.  One launch / two, us: tokens given, 16 requests of 32000 values 11.5 / 12.8,
// of 40000 13.2 / 12.8, of 50000 15.2 / 12.8, of 65000 15.1 / 12.8; drawn, 16 of 32000 10.0 / 11.9 without further sums and
// 15.3 / 17.3 with one, of 40000 11.1 / 11.8 and 15.4 / 14.8, of 65000 12.3 / 11.6 and 17.6 / 14.9.  A launch takes some 3 us of
// the host's time besides.
constexpr int kSumFrom = 40960;

// Workgroups per row of scores, where there are fewer rows than fill the card, of at least four rounds of loads.  Of up to
// 512 / 768 / 1024 in all, us of both launches over rows of 100003 bf16 values: 100 rows 7.6 / 7.9 / 8.1, 150 9.7 / 8.9 / 9.2,
// 464 19.7 / 19.6 / 21.0, 512 21.1 / 21.3 / 22.9; 300 rows of 32000 fp16 ones 8.6 / 7.3 / 7.5.
int row_shares(const VerifyArgs& a) {
  const int64_t most = ((int64_t)a.vocab + 4 * kBestStep - 1) / (4 * kBestStep);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, 768 / std::max(a.tokens_count, 1)));
}

template <class T>
void best_launch(const VerifyArgs& a, int shares, hipStream_t stream) {
  const int part = (int)((((int64_t)a.vocab + shares - 1) / shares + kBestStep - 1) / kBestStep * kBestStep);
  best_token_kernel<T><<<a.tokens_count * shares, kBestThreads, 0, stream>>>(a, shares, part);
}

// Pieces of a row whose sums a launch of their own leaves; 0: one workgroup adds the row up.
int summed_pieces(const VerifyArgs& a) { return a.vocab <= kSumFrom ? 0 : (a.vocab + kPiece - 1) / kPiece; }

// Workgroups that add up a request's row again together, four pieces at a time; no more in all than the card has CUs, one for
// each.  In all up to 128 / 256 / 512, us of both launches over rows of 150001 values: 16 requests 17.5 / 15.3 / 15.4, 32
// 24.4 / 22.4 / 24.9, 64 49.6 / 45.6 / 45.8; without such sums the same to 0.2.
int pick_team(const VerifyArgs& a, int pieces) {
  return pieces > kPickThreads ? 1 : std::max(1, std::min((pieces + 3) / 4, 256 / a.seqs));
}

template <bool DRAWN>
hipError_t sample_launch(const VerifyArgs& a, hipStream_t stream) {
  const int pieces = summed_pieces(a);
  if (pieces) {
    verify_sum_kernel<DRAWN><<<dim3(pieces, a.seqs), kSumThreads, 0, stream>>>(a, pieces);
    if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  }
  verify_pick_kernel<DRAWN><<<dim3(a.seqs, DRAWN ? pick_team(a, pieces) : 1), kPickThreads, 0, stream>>>(a, pieces);
  return hipGetLastError();
}

}  // namespace

hipError_t draft_trees_launch(const DraftTreesArgs& a, hipStream_t stream) {
  draft_trees_kernel<<<(a.seqs + kTreeWaves - 1) / kTreeWaves, 64 * kTreeWaves, 0, stream>>>(a);
  return hipGetLastError();
}

size_t verify_workspace_bytes(const VerifyArgs& a) {
  if (a.mode == kVerifyBest) return (size_t)a.tokens_count * row_shares(a) * sizeof(uint64_t);
  const size_t sums = (size_t)a.seqs * summed_pieces(a) * sizeof(double);
  return a.mode == kVerifyDrawn && sums ? 2 * sums + a.seqs * sizeof(uint32_t) : sums;
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
