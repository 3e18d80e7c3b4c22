// Attention of few rows per request over the pages of a cache: decode steps, short continuations.
//
//   out[t, h] = sum_s softmax_s(scale q[t, h] . k[s, kv]) v[s, kv],   s <= position of t,   kv = h / rep
//
// or, where the new tokens are the nodes of a tree (TREE), over the s before them and the node's ancestors.
//
// What bounds it: the bytes of K and V, read once.  Three requests of up to 131071 tokens (8 KV heads of 128) take 204 us,
// 6.3 TB/s of the 7.1 that a plain read of the card reaches; 64 of 100 .. 8191 tokens (2 of 128), 112 MB, take 25 us: 21 the
// first launch, of which 15.8 at that rate, the rest finding the stretches until the first keys are there, and 4 the second.
// LDS bank conflicts are 27% of its LDS cycles there, which bound nothing: the vector pipe is busy 13% of the time.  So the
// work of all requests is laid end to end, in units of 32 keys a wavefront of one item (request, row tile, KV head), and cut
// into one equal stretch per workgroup whatever the lengths are; a workgroup finds its stretch from the lengths by itself
// (they are read on the device only, so a captured launch follows them).  The wavefronts of a workgroup take 32 keys each
// and do not wait for each other: each keeps its keys' tiles of K and V coming through LDS buffers of its own by
// asynchronous copies, and they meet at the end of an item.  An item inside one stretch is finished there; the pieces of
// one that is cut go to the workspace (maximum, sum, unscaled outputs, 32 bits) and a second launch joins them, in the
// order of the keys: results do not depend on timing.
#pragma once

#include "kf_attn_tiles.h"

namespace kf {
namespace {

// Beginning and ending an item takes about as long as these many units: they count for it when the work is cut, or
// workgroups with many short items would be the last ones.  With 0, 1, 2, 3: 39.6, 28.4, 25.6, 25.1 us for 64 requests of
// 100 .. 8191 tokens (2 KV heads of 128), 58.6, 45.6, 41.7, 41.7 for 128 of 50 .. 900 (8 of 128, four wavefronts).
constexpr int kFewItem = 2;

template <int HDP_, int MT_, int WAVES_, int STAGES_ = HDP_ == 64 ? 4 : 2>
struct FewConfig {
  static constexpr int HDP = HDP_, MT = MT_;
  static constexpr int WAVES = WAVES_;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int STAGES = STAGES_;
  static constexpr int ROW = HDP * 2;
  static constexpr int STAGE = 2 * 32 * ROW;         // K and V of 32 keys
  static constexpr int RING = STAGES * STAGE;        // of one wavefront
  static constexpr int ROWS = 16 * MT;
  static constexpr int UNIT = 32 * WAVES;            // keys
  static constexpr int LDS = WAVES * RING;           // 32 KiB a wavefront as a rule, half or more of it on its way
  static_assert(WAVES * ROWS * HDP * 4 <= LDS, "the wavefronts' sums meet in the buffers");
};

// A request's items, (row tiles) x (KV heads), each of *key_units units of keys (one at least, so that every row is
// written); what one item counts is item_cost: its units and ITEM, or 1 where items are not cut.
template <class C>
__device__ __forceinline__ int few_items(const AttnArgs& a, int s, int rep, int max_rows, int* key_units) {
  const int rows = max(seq_offset(a.cu, s + 1, a.seqs, a.tokens) - seq_offset(a.cu, s, a.seqs, a.tokens), 0) * rep;
  *key_units = max((seq_keys<true>(a, s, 0).keys + C::UNIT - 1) / C::UNIT, 1);
  return rows > max_rows ? 0 : (rows + C::ROWS - 1) / C::ROWS * a.kv_heads;
}
template <class C, bool CUT>
__device__ __forceinline__ int item_cost(int key_units) {
  return CUT ? key_units + kFewItem : 1;
}

__device__ __forceinline__ float max_groups(float v) {  // of lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto s = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return max_halves(fmaxf(bit_cast<float>((uint32_t)s[0]), bit_cast<float>((uint32_t)s[1])));
}
__device__ __forceinline__ float add_groups(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return add_halves(bit_cast<float>((uint32_t)s[0]) + bit_cast<float>((uint32_t)s[1]));
}

template <class C>
struct FewShared {
  __attribute__((aligned(1024))) unsigned char smem[C::LDS];
  float stat[2][C::WAVES][C::ROWS];
  int scan[C::WAVES], found[2];
};

// Stretch `me` of `stretches`, by one workgroup.
// CUT: items may be cut; otherwise every stretch is of whole ones, and nothing is left to join.
template <class E, class C, bool CUT, bool TREE>
__device__ __forceinline__ void few_rows_stretch(const AttnArgs& args, FewShared<C>& sh, int me, int stretches, int rep,
                                                 int max_rows, float scale_log2, float* ws, Piece* pieces) {
  constexpr int HDP = C::HDP, MT = C::MT;
  using Copy = TileCopy<E, HDP, true>;
  constexpr int PER_STAGE = 4 * Copy::N, ROW = C::ROW;  // copy instructions of a stage
  constexpr int ST = HDP / 32, DT = HDP / 16;
  unsigned char* const smem = sh.smem;
  auto& stat = sh.stat;
  auto& scan = sh.scan;
  auto& found = sh.found;
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  int begin, end, per;
  {
    const AttnArgs& a = args;
    // This workgroup's stretch.  Every thread sums a run of requests; the one whose run holds the stretch's
    // first unit says which request that is.
    const int run = (a.seqs + C::THREADS - 1) / C::THREADS;
    const int s0 = min(tid * run, a.seqs), s1 = min(s0 + run, a.seqs);
    int ku, mine = 0;
    for (int s = s0; s < s1; ++s) {
      const int n = few_items<C>(a, s, rep, max_rows, &ku);
      mine = add_work(mine, n * item_cost<C, CUT>(ku));
    }
    const int upto = work_prefix(mine);
    if (lane == 63) scan[wave] = upto;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < C::WAVES; ++w) {
      if (w < wave) before = add_work(before, scan[w]);
      total = add_work(total, scan[w]);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (total == kNoWork) total = 0;
    per = total / stretches + (total % stretches ? 1 : 0);
    const Stretch stretch = stretch_of(total, per, me);
    begin = stretch.begin, end = stretch.end;
    if (stretch.begins_in(before, mine)) {
      int at = before;
      for (int s = s0; s < s1; ++s) {
        const int n = few_items<C>(a, s, rep, max_rows, &ku) * item_cost<C, CUT>(ku);
        if (begin < at + n) {
          found[0] = s;
          found[1] = at;
          break;
        }
        at += n;
      }
    }
    if (CUT && tid == 0) pieces[me].seq = -1;
    __syncthreads();

    // Rows in no sequence.
    if (a.zero_rest) {
      const int t0 = seq_offset(a.cu, a.seqs, a.seqs, a.tokens);
      const int cpr = a.head_dim / 8, per_row = a.heads * cpr;
      for (int64_t i = (int64_t)me * C::THREADS + tid; i < (int64_t)(a.tokens - t0) * per_row;
           i += (int64_t)stretches * C::THREADS) {
        const int64_t t = i / per_row;
        const int r = (int)(i - t * per_row), h = r / cpr;
        *(u32x4*)((E*)a.out + (t0 + t) * a.out_token + h * a.out_head + 8 * (r - h * cpr)) = u32x4{0, 0, 0, 0};
      }
    }
    if (begin >= end || found[0] < 0) return;
  }

  int seq = __builtin_amdgcn_readfirstlane(found[0]);
  int seq_at = __builtin_amdgcn_readfirstlane(found[1]);  // the request's first unit
  const uint32_t ring = lds + (uint32_t)wave * C::RING;
  const uint32_t k_at = (uint32_t)l16 * ROW + 16u * (uint32_t)(g ^ swizzle_k<HDP>(l16));
  const int vrow = 4 * g + (l16 >> 2);
  const uint32_t v_at = 32u * ROW + (uint32_t)vrow * ROW + 16u * (uint32_t)(((l16 & 3) >> 1) ^ swizzle_v16<HDP>(vrow)) +
                        8u * (uint32_t)(l16 & 1);
  const float slack = 8.0f / scale_log2;
  for (int at = begin; at < end;) {
    const AttnArgs a = reload_args();
    const Copy copy(a.k_token, a.v_token, a.head_dim, lane);
    int n, ku;
    while ((n = few_items<C>(a, seq, rep, max_rows, &ku) * item_cost<C, CUT>(ku)) <= at - seq_at) {  // next request with items
      seq_at += n;
      if (++seq >= a.seqs) return;
    }
    const int cost = item_cost<C, CUT>(ku), item = (at - seq_at) / cost, item_at = seq_at + item * cost;
    // The stretch's part of the item; of what it counts, the beginning comes first.
    const int first_unit = item_at + (CUT ? kFewItem : 0);
    const int u0 = CUT ? max(at - first_unit, 0) : 0, u1 = CUT ? min(ku, end - first_unit) : ku;
    at = item_at + cost;
    if (u1 <= u0) break;  // not even its first unit
    const int kv = item % a.kv_heads, row0 = item / a.kv_heads * C::ROWS;
    const int tok0 = seq_offset(a.cu, seq, a.seqs, a.tokens);
    const int len = seq_offset(a.cu, seq + 1, a.seqs, a.tokens) - tok0, rows = len * rep;
    const SeqKeys sk = seq_keys<true>(a, seq, len);
    const int64_t table_at = (int64_t)seq * a.table_stride;

    u32x4 qf[MT][ST];
    int limit[MT];     // the row's last key
    TreeRow node[MT];  // TREE: its keys
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = min(row0 + 16 * t + l16, rows - 1), tok = row / rep, head = kv * rep + (row - tok * rep);
      if constexpr (TREE) node[t].bits = a.ancestors[tok0 + tok];
      else limit[t] = sk.last_key(tok);
      const E* const qp = (const E*)a.q + (size_t)(tok0 + tok) * a.q_token + (size_t)head * a.q_head;
#pragma unroll
      for (int s = 0; s < ST; ++s)
        qf[t][s] = 4 * s + g < a.head_dim / 8 ? load_global16(qp + 32 * s + 8 * g) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) arrived(qf[t]);
    // Keys of the tile's last row, the last that all its rows attend to.
    const int kend = TREE ? sk.keys : sk.last_key(min(row0 + C::ROWS - 1, rows - 1) / rep) + 1;
    const int first_limit = TREE ? sk.before() - 1 : sk.last_key(row0 / rep);

    auto page_of = [&](int key) {  // uniform; -1: not in the cache
      if (kend <= 0) return -1;
      const int p = load_const(a.table, table_at + (min(key, kend - 1) >> a.log2_block));
      return (unsigned)p < (unsigned)a.num_pages ? p : -1;
    };
    auto issue = [&](int i, int p0, int p1) {  // unit u0 + i; pages of its two 16 keys
      const int key0 = (u0 + i) * C::UNIT + 32 * wave;
      const uint32_t dst = ring + (uint32_t)(i % C::STAGES) * C::STAGE;
      const E* const k = (const E*)a.k + kv * a.k_head;
      const E* const v = (const E*)a.v + kv * a.v_head;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int page = half ? p1 : p0, key = key0 + 16 * half;
        const int slot = key & ((1 << a.log2_block) - 1);
        copy(dst + (16 * half) * ROW, dst + (32 + 16 * half) * ROW, k + page * a.k_page + slot * a.k_token,
             v + page * a.v_page + slot * a.v_token, page >= 0 ? kend - key : 0, lane);
      }
    };

    float4_t o[MT][DT];
    float m[MT], mc[MT], sum[MT], limit_max[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m[t] = limit_max[t] = -__builtin_inff();
      mc[t] = sum[t] = 0.0f;
#pragma unroll
      for (int c = 0; c < DT; ++c) o[t][c] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int n_units = u1 - u0, live_rows = rows - row0;
    auto key_of = [&](int i) { return (u0 + i) * C::UNIT + 32 * wave; };
    int next0 = page_of(key_of(0)), next1 = page_of(key_of(0) + 16);
    for (int i = 1 - C::STAGES; i < n_units; ++i) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer's last reads are done
      const bool more = i + C::STAGES - 1 < n_units;
      if (more) {
        issue(i + C::STAGES - 1, next0, next1);
        next0 = page_of(key_of(i + C::STAGES)), next1 = page_of(key_of(i + C::STAGES) + 16);
      }
      if (i < 0) continue;
      if (more) wait_vmcnt<PER_STAGE * (C::STAGES - 1)>();
      else wait_vmcnt<0>();
      const int key0 = key_of(i);
      if (key0 >= kend) continue;
      const uint32_t buf = ring + (uint32_t)(i % C::STAGES) * C::STAGE;

      const bool bad0 = page_of(key0) < 0, bad1 = page_of(key0 + 16) < 0;
      const bool masked = key0 + 31 > first_limit || bad0 || bad1;
      // The last of this lane's keys key0 + 16 u + 4 g + (0 .. 3) that its row attends to, as 0 .. 3 (below: none).
      auto keys_at = [&](int t, int u) { return (u ? bad1 : bad0) ? -1 : limit[t] - (key0 + 16 * u + 4 * g); };
      u32x4 p[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        p[t] = u32x4{0, 0, 0, 0};
        if (MT > 1 && 16 * t >= live_rows) continue;
        float4_t s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int st = 0; st < ST; ++st)
            s[u] = Elem<E>::mfma16(lds_read16(((buf + k_at) ^ (uint32_t)(64 * st)) + u * 16 * ROW), qf[t][st], s[u]);
        }
        if (masked) {
          uint32_t seen = 0;  // this lane's keys: bits 16 u + e
          if constexpr (TREE)
            seen = ((uint32_t)node[t].from(sk, key0) & ((bad0 ? 0 : 0xFFFF) | (bad1 ? 0 : 0xFFFF0000u))) >> (4 * g);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if constexpr (TREE) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(seen >> (16 * u + e) & 1)) s[u][e] = -__builtin_inff();
            } else {
              const int last = keys_at(t, u);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (e > last) s[u][e] = -__builtin_inff();
            }
          }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_groups(mx);
        if (__builtin_expect(__ballot(mx > limit_max[t]) != 0, 0)) {
          const float mn = fmaxf(m[t], mx);
          const float mcn = mn == -__builtin_inff() ? 0.0f : mn * scale_log2;
          const float f = m[t] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mc[t] - mcn);
          m[t] = mn;
          mc[t] = mcn;
          limit_max[t] = mn + slack;
          sum[t] *= f;
#pragma unroll
          for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][c][e] *= f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], scale_log2, -mc[t]));
            sum[t] += s[u][e];
          }
          p[t][2 * u] = Elem<E>::pack(s[u][0], s[u][1]);
          p[t][2 * u + 1] = Elem<E>::pack(s[u][2], s[u][3]);
        }
      }
      auto v_block = [&](int c) {
        const uint32_t va = (buf + v_at) ^ (uint32_t)(32 * c);
        const u32x2 v0 = lds_read_tr(va), v1 = lds_read_tr(va + 16 * ROW);
        return u32x4{v0[0], v0[1], v1[0], v1[1]};
      };
      const uint32_t v_tile = buf + 32 * ROW;
      if (__builtin_expect(masked, 0) && lds_any_nonfinite<E>(v_tile, 32 * ROW / 1024, lane)) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int c = 0; c < DT; ++c) {
            float4_t add = {0.0f, 0.0f, 0.0f, 0.0f};  // of dims 16 c + 4 g + (0 .. 3)
#pragma unroll 1
            for (int k = 0; k < 32; ++k)
              if ((TREE ? node[t].sees(sk, key0 + k) : key0 + k <= limit[t]) && !(k >> 4 ? bad1 : bad0))
                add += nonfinite_of<E>(
                    lds_read8(v_tile + k * ROW + 16 * ((2 * c + (g >> 1)) ^ swizzle_v16<HDP>(k)) + 8 * (g & 1)));
            o[t][c] += add;
            // Here, not for all tiles at the end: this rare path takes no registers from the others.
            asm volatile("" : "+v"(o[t][c]));
          }
        lds_finite_only<E>(v_tile, 32 * ROW / 1024, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int c = 0; c < DT; ++c) {
        const u32x4 v = v_block(c);
#pragma unroll
        for (int t = 0; t < MT; ++t)
          if (MT == 1 || 16 * t < live_rows) o[t][c] = Elem<E>::mfma16(v, p[t], o[t][c]);
      }
    }

    // The wavefronts' maxima, sums and outputs meet in the buffers.
    __syncthreads();  // every wavefront has read its last tile
    const AttnArgs b = reload_args();
    float* const acc = reinterpret_cast<float*>(smem);  // [WAVES][ROWS][HDP]
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const float total_sum = add_groups(sum[t]);
      if (g == 0) {
        stat[0][wave][16 * t + l16] = m[t] == -__builtin_inff() ? m[t] : mc[t];
        stat[1][wave][16 * t + l16] = total_sum;
      }
      if (16 * t + l16 < live_rows) {
#pragma unroll
        for (int c = 0; c < DT; ++c)
          *reinterpret_cast<float4_t*>(acc + (wave * C::ROWS + 16 * t + l16) * HDP + 16 * c + 4 * g) = o[t][c];
      }
    }
    __syncthreads();
    const bool whole = !CUT || (u0 == 0 && u1 == ku);
    const int part = 2 * me + (u0 == 0 ? 1 : 0);
    float* const part_o = ws + (size_t)part * C::ROWS * (HDP + 2);
    float* const part_s = part_o + C::ROWS * HDP;
    for (int i = tid; i < min(live_rows, C::ROWS) * (HDP / 4); i += C::THREADS) {
      const int r = i / (HDP / 4), d = 4 * (i % (HDP / 4));
      float top = stat[0][0][r];
#pragma unroll
      for (int w = 1; w < C::WAVES; ++w) top = fmaxf(top, stat[0][w][r]);
      float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < C::WAVES; ++w) {
        // A wavefront without keys for the row has m = -inf, sums of 0 and no part (0 here, not -inf - -inf).
        const float f = stat[0][w][r] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(stat[0][w][r] - top);
        const float4_t x = *reinterpret_cast<const float4_t*>(acc + (w * C::ROWS + r) * HDP + d);
        // A NaN among a wavefront's scores is in its sum, whatever its maximum says.
        l += stat[1][w][r] != stat[1][w][r] ? stat[1][w][r] : f * stat[1][w][r];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += scaled(x[e], f);
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no keys: zeros
        const int row = row0 + r, tok = row / rep, head = kv * rep + (row - tok * rep);
        if (d < b.head_dim)
          store_global((E*)b.out + (size_t)(tok0 + tok) * b.out_token + (size_t)head * b.out_head + d,
                       u32x2{Elem<E>::pack(v[0] * inv, v[1] * inv), Elem<E>::pack(v[2] * inv, v[3] * inv)});
      } else {
        *reinterpret_cast<float4_t*>(part_o + r * HDP + d) = v;
        if (d == 0) {
          part_s[r] = top;
          part_s[C::ROWS + r] = l;
        }
      }
    }
    if (tid == 0 && u0 == 0 && !whole)
      pieces[me] = Piece{seq, row0, kv, last_stretch(item_at, cost, per)};
    __syncthreads();  // the sums have been read: the buffers are free
  }
}

}  // namespace
}  // namespace kf
