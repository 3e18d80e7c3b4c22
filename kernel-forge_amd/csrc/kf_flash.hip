// Causal attention of packed sequences with many rows per sequence, over contiguous keys (whole prompts) or over
// the pages of a cache (chunks of prompts): one pass over the keys with the running maximum and sum of the softmax.
//
//   out[t, h] = sum_s softmax_s(scale q[t, h] . k[s, kv]) v[s, kv],   s <= position of t,   kv = h / rep
//
// or, over pages, where the new tokens are the nodes of a tree, over the s before them and the node's ancestors.
//
// A workgroup owns 128 rows of one KV head (kf_attn_tiles.h), 32 per wavefront, and walks their keys 64 at a time (32
// for heads of more than 128, whose outputs fill half the registers) through two LDS buffers.  Scores, maximum, sum
// and outputs are held in 32 bits; probabilities are rounded to the inputs' type for the second matrix product (half
// a step of that type, as inputs are), the outputs once more when they are stored.  The maximum that the exponentials
// are taken against follows the true one only when it is exceeded by a factor 2^8: outputs and sums are then
// rescaled, which most tiles after the first spare.
//
// What bounds it: a tile of 64 keys costs a wavefront 16 (64 dims) or 32 (128 dims) matrix instructions of 32 cycles
// and some 150 vector instructions for the softmax of its 32 x 64 scores, 32 of them exponentials, which take two slots.
// With 64 dims the vector pipe leads: 16001 tokens of 32 heads take 1.11 ms, 950 TFLOP/s, vector pipe busy 89% of the
// CUs' cycles, matrix cores 58%, no LDS bank conflicts, the clock at 1.64 GHz.  With 128 dims neither is full, at two
// wavefronts per SIMD: 8000 tokens of 32 heads take 0.49 ms, 1070 TFLOP/s, matrix cores 55%, vector pipe 48%, of 1190 ..
// 1630 TFLOP/s that matrix products of 4096 .. 16384 reach on the card.  Tried without gain: the next tile's scores
// computed while a tile's exponentials are (0.50 .. 0.52 ms), tiles of 32 keys (0.49 ms; 16 ragged prompts 55 us, not
// 49).  A batch of a few hundred row tiles waits for its longest: 16 prompts of 19 .. 1455 tokens (12 heads on 2 of 128)
// take 45 .. 49 us, the longest row tile 23 tiles of keys where the work spread evenly is 14.
#include <math.h>

#include <algorithm>

#include "kf_few_rows.h"
#include "kf_launch.h"

namespace kf {
namespace {

constexpr int kFlashWaves = 4, kFlashThreads = 64 * kFlashWaves;
constexpr int kFlashRows = 32 * kFlashWaves;

// Wavefronts per SIMD that the registers have to allow: one computes scores while another works on its
// softmax.  From two on the products also accumulate in ordinary registers, without moves.
// The kernel that cuts the work needs some registers more.
constexpr int flash_waves_per_simd(int hdp, bool cut) { return hdp == 64 ? (cut ? 3 : 4) : hdp == 128 ? 2 : 1; }

// Where the keys are: rows beside the queries' own, or pages of a cache; over pages the new tokens are a chain or a tree.
enum class Keys { kPacked, kPages, kTree };

// Two groups where their buffers fit.
constexpr int flash_groups(int hdp) { return hdp == 256 ? 1 : 2; }

template <int HDP>
struct FlashConfig {
  static constexpr int ROW = HDP * 2;  // bytes
  static constexpr int KEYS = HDP == 256 ? 32 : 64;
  static constexpr int TILE = KEYS * ROW;
  // Queries of more than 128 dims leave no registers for themselves beside the outputs: each lane's stay in LDS.
  static constexpr bool Q_LDS = HDP == 256;
  static constexpr int LDS = 4 * TILE + (Q_LDS ? kFlashRows * ROW : 0);
};
// GROUPS of four wavefronts work on the same rows, each on every GROUPS-th tile of keys, and join at the end: where
// there are fewer row tiles than the GPU holds workgroups, an item then ends sooner.
template <int HDP, int GROUPS>
struct FlashShared {
  __attribute__((aligned(1024))) unsigned char smem[GROUPS * FlashConfig<HDP>::LDS];
  int found[2][GROUPS * kFlashWaves];  // infinities or NaN in a masked tile
  int patch_from;
  float stat[GROUPS > 1 ? 2 * 64 * kFlashWaves : 1];
};

// Rows row0 .. + 127 of a sequence over its key tiles tile0 .. tiles - 1 (those that it has of them).
// tok0, len, sk: the sequence's new tokens and keys.  part: nullptr, or where the maximum, sum and unscaled outputs of an
// item that is cut go: rows of values, for trees as the lanes hold them.
template <class E, int HDP, Keys KEYS_OF, int GROUPS>
__device__ __forceinline__ void flash_item(const AttnArgs& a, FlashShared<HDP, GROUPS>& sh, int rep, float scale_log2, int seq,
                                           int tok0, int len, SeqKeys sk, int row0, int kv, int tile0, int tiles, float* part) {
  using C = FlashConfig<HDP>;
  constexpr bool PAGED = KEYS_OF != Keys::kPacked, TREE = KEYS_OF == Keys::kTree;
  constexpr int ROW = C::ROW, KEYS = C::KEYS, KU = KEYS / 32, KK = KEYS / 16, TILE = C::TILE;
  constexpr int MINE = KEYS / kFlashWaves;          // keys of a tile that a wavefront fetches
  constexpr int ST = HDP / 16;                      // k steps of the first product
  constexpr int DT = HDP / 32;                      // 32-row tiles of O^T
  constexpr bool Q_LDS = C::Q_LDS;
  auto& found = sh.found;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % kFlashWaves);
  const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  unsigned char* const smem = sh.smem + group * C::LDS;
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int rows = len * rep;

  // This lane's row.  Rows past the end repeat the last one and are not stored.
  const int my_row = row0 + 32 * wave + (lane & 31);
  const int row = min(my_row, rows - 1);
  const int tok = row / rep;
  const int head = kv * rep + (row - tok * rep);
  // Keys: positions before this lane's row's own, itself included.
  const int limit = sk.last_key(tok);  // may be negative: no keys
  TreeRow node;
  if constexpr (TREE) node.bits = a.ancestors[tok0 + tok];
  const int wave_row = row0 + 32 * wave;
  const int wave_lo = TREE ? sk.before() - 1 : sk.last_key(min(wave_row, rows - 1) / rep);
  const int wave_hi = TREE ? sk.keys - 1 : sk.last_key(min(wave_row + 31, rows - 1) / rep);
  const int first_limit = TREE ? sk.before() - 1 : sk.last_key(row0 / rep);  // the last key that all rows attend to
  const int kend = TREE ? sk.keys : sk.last_key(min(row0 + kFlashRows - 1, rows - 1) / rep) + 1;
  tiles = min(tiles, kend <= 0 ? 0 : (kend + KEYS - 1) / KEYS);
  const int mine0 = tile0 + group;  // this group's first tile

  // The pages of the groups' next tiles come by one vector load, lane i's those of 16 keys, a tile ahead of the copies; the first
  // ones beside the queries.
  const int* const table = a.table + (PAGED ? (int64_t)seq * a.table_stride : 0);
  auto load_pages = [&](int kt0) {
    const int key = kt0 * KEYS + 16 * (lane % (GROUPS * KK));
    const int p = load_const(table, min(key, kend - 1) >> a.log2_block);
    return (unsigned)p < (unsigned)a.num_pages ? p : -1;  // -1: not in the cache
  };
  int pages = 0;
  if constexpr (PAGED)
    if (tile0 < tiles) pages = load_pages(tile0);

  u32x4 qf[Q_LDS ? 1 : ST];
  u32x4* const q_lds = reinterpret_cast<u32x4*>(smem + 4 * TILE) + wave * ST * 64 + lane;
  {
    const E* const qp = (const E*)a.q + (size_t)(tok0 + tok) * a.q_token + (size_t)head * a.q_head;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      const u32x4 x = 2 * s + half < a.head_dim / 8 ? load_global16(qp + 16 * s + 8 * half) : u32x4{0, 0, 0, 0};
      if constexpr (Q_LDS) q_lds[64 * s] = x;
      else qf[s] = x;
    }
    arrived(qf);
  }

  // Copies.  A wavefront fetches rows 16 wave .. + 15 of both tiles: one page, as pages hold 16 keys at least.
  const TileCopy<E, HDP, false, MINE> copy(a.k_token, a.v_token, a.head_dim, lane, MINE * wave);
  auto issue = [&](int kt, uint32_t buf, int page) {
    const int key0 = kt * KEYS + MINE * wave;
    const E* const k = (const E*)a.k + kv * a.k_head;
    const E* const v = (const E*)a.v + kv * a.v_head;
    const uint32_t dst = lds + buf + (uint32_t)(MINE * wave) * ROW;
    if constexpr (PAGED) {
      const int slot = key0 & ((1 << a.log2_block) - 1);
      copy(dst, dst + TILE, k + page * a.k_page + slot * a.k_token, v + page * a.v_page + slot * a.v_token,
           page >= 0 ? kend - key0 : 0, lane);
    } else {
      copy(dst, dst + TILE, k + (int64_t)(tok0 + key0) * a.k_token, v + (int64_t)(tok0 + key0) * a.v_token, kend - key0,
           lane);
    }
  };

  float16_t o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
  float m = -__builtin_inff();       // the maximum that the exponentials are taken against
  float mc = 0.0f, sum = 0.0f;       // m in units of the exponent (0 while there is none), this lane's sum
  float limit_max = -__builtin_inff();
  const float slack = 8.0f / scale_log2;

  // Reads of the tiles: K rows lane % 32, V blocks as transposing reads want them.
  const uint32_t k_at = (uint32_t)(lane & 31) * ROW + 16u * (uint32_t)(half ^ swizzle_k<HDP>(lane & 31));
  const int vrow = 4 * half + ((lane >> 2) & 3);
  const uint32_t v_at = (uint32_t)vrow * ROW +
                        16u * (uint32_t)((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle_v<HDP>(vrow)) +
                        8u * (uint32_t)(lane & 1) + TILE;

  int patch_from = 0x7fffffff;  // first key of a tile with masks whose infinities and NaN were taken out
  // Which of this wavefront's pages and of all groups' are not there, now and in the next tiles.
  uint64_t missing = 0, next_missing = 0;
  auto my_page = [&] { return __builtin_amdgcn_readlane(pages, group * KK + MINE * wave / 16); };
  auto none = [&] { return __ballot(pages < 0) & ((1u << (GROUPS * KK)) - 1); };
  if (tile0 < tiles) {
    if constexpr (PAGED) next_missing = none();
    if (mine0 < tiles) issue(mine0, 0, PAGED ? my_page() : 0);
    if constexpr (PAGED) pages = load_pages(tile0 + GROUPS);
  }
  uint32_t buf = 2 * TILE;
  for (int kt0 = tile0; kt0 < tiles; kt0 += GROUPS) {  // the groups' iterations and barriers are the same
    const int kt = kt0 + group;
    buf ^= 2 * TILE;
    dma_barrier();
    missing = next_missing;
    if constexpr (PAGED) next_missing = none();
    const int page = PAGED ? my_page() : 0;
    if constexpr (PAGED) pages = load_pages(kt0 + 2 * GROUPS);  // before the copies: the wait for them is a wait for it
    if (kt + GROUPS < tiles) issue(kt + GROUPS, 2 * TILE - buf, page);
    const int key0 = kt * KEYS;

    // Masks: keys past a row's own, pages that are not there (bit i of `bad`: keys key0 + 16 i .. + 15).
    const uint32_t bad = (uint32_t)(missing >> (group * KK)) & ((1u << KK) - 1);
    const uint32_t my_v = lds + buf + TILE + (uint32_t)(MINE * wave) * ROW;  // the rows of V that this wavefront looks after
    // The same in all wavefronts: some group's tile has masks.
    if (__builtin_expect((kt0 + GROUPS) * KEYS - 1 > first_limit || missing != 0, 0)) {
      const int flag = (buf != 0) ? 1 : 0;
      const bool any = kt < tiles && lds_any_nonfinite<E>(my_v, MINE * ROW / 1024, lane);
      if (lane == 0) found[flag][group * kFlashWaves + wave] = any;
      lds_barrier();
      bool some = false, mine = false;
#pragma unroll
      for (int w = 0; w < GROUPS * kFlashWaves; ++w) {
        some |= found[flag][w] != 0;
        mine |= w / kFlashWaves == group && found[flag][w] != 0;
      }
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(some), 0)) {
        if (__builtin_amdgcn_readfirstlane(mine)) {
          lds_finite_only<E>(my_v, MINE * ROW / 1024, lane);
          patch_from = min(patch_from, key0);
        }
        lds_barrier();
      }
    }
    if (key0 > wave_hi || kt >= tiles) continue;  // only other wavefronts have keys here

    float16_t s[KU];
    const uint32_t kb = lds + buf + k_at;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
    // This wavefront's matrix products go before the other wavefronts' softmax: their results are waited for longest.
    // (8000 tokens of 32 heads of 128: 507 -> 497 us; 64 dims and short prompts the same without.)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int u = 0; u < KU; ++u)
        s[u] = Elem<E>::mfma32(lds_read16((kb ^ (uint32_t)(32 * st)) + u * 32 * ROW),
                               Q_LDS ? q_lds[64 * st] : qf[Q_LDS ? 0 : st], s[u]);

    __builtin_amdgcn_s_setprio(0);
    const bool masked = key0 + KEYS - 1 > wave_lo || bad != 0;
    // The last of this lane's keys key0 + 8 q + 4 half + (0 .. 3) that its row attends to, as 0 .. 3 (below: none).
    auto keys_at = [&](int q) { return (bad >> (q >> 1)) & 1 ? -1 : limit - (key0 + 8 * q + 4 * half); };
    const uint32_t vb = lds + buf + v_at;
    auto v_block = [&](int kk, int t) {
      const uint32_t at = (vb ^ (uint32_t)(64 * t)) + kk * 16 * ROW;
      const u32x2 v0 = lds_read_tr(at), v1 = lds_read_tr(at + 8 * ROW);
      return u32x4{v0[0], v0[1], v1[0], v1[1]};
    };
    if (__builtin_expect(masked, 0)) {
      uint64_t seen = 0;  // this lane's keys: bits 8 q + e
      if constexpr (TREE) {
        uint64_t there = 0;
#pragma unroll
        for (int i = 0; i < KK; ++i) there |= (bad >> i) & 1 ? 0 : 0xFFFFull << (16 * i);
        seen = (node.from(sk, key0) & there) >> (4 * half);
      }
#pragma unroll
      for (int q = 0; q < 2 * KK; ++q) {
        if constexpr (TREE) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((uint32_t)(seen >> (32 * (q >> 2))) >> (8 * (q & 3) + e) & 1)) s[q >> 2][4 * (q & 3) + e] = -__builtin_inff();
        } else {
          const int last = keys_at(q);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e > last) s[q >> 2][4 * (q & 3) + e] = -__builtin_inff();
        }
      }
    }

    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * KU; ++i) mx = fmaxf(mx, s[i >> 4][i & 15]);
    mx = max_halves(mx);
    if (__builtin_expect(__ballot(mx > limit_max) != 0, 0)) {
      const float mn = fmaxf(m, mx);
      const float mcn = mn == -__builtin_inff() ? 0.0f : mn * scale_log2;
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mc - mcn);
      m = mn;
      mc = mcn;
      limit_max = mn + slack;
      sum *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= f;
    }
    u32x4 p[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[kk >> 1][8 * (kk & 1) + i], scale_log2, -mc));
        sum += e[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) p[kk][i] = Elem<E>::pack(e[2 * i], e[2 * i + 1]);
      asm volatile("" : "+v"(sum), "+v"(p[kk]));  // summed and rounded here: the 32-bit probabilities are not kept
    }

#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] = Elem<E>::mfma32(v_block(kk, t), p[kk], o[t]);
  }

  sum = add_halves(sum);
  if constexpr (GROUPS > 1) {
    // The second group's outputs, maxima and sums go through the buffers to the first one.
    static_assert(GROUPS == 2, "one joins the other");
    const int t256 = 64 * wave + lane;
    if (threadIdx.x == 0) sh.patch_from = 0x7fffffff;
    lds_barrier();  // the tiles have been read
    float4_t* const acc = reinterpret_cast<float4_t*>(sh.smem);  // [4 DT][256]
    if (group == 1) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[(4 * t + i) * 256 + t256] = float4_t{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
      sh.stat[t256] = m;
      sh.stat[256 + t256] = sum;
      if (lane == 0 && patch_from != 0x7fffffff) atomicMin(&sh.patch_from, patch_from);
    }
    lds_barrier();
    if (group == 1) return;
    const float m1 = sh.stat[t256], mn = fmaxf(m, m1);
    const float mcn = mn == -__builtin_inff() ? 0.0f : mn * scale_log2;
    const float f0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mc - mcn);
    const float f1 = m1 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m1 * scale_log2 - mcn);
    // A NaN among a group's scores is in its sum, whatever its maximum says; without a maximum the others are zeros.
    const float s1 = sh.stat[256 + t256];
    sum = (sum != sum ? sum : f0 * sum) + (s1 != s1 ? s1 : f1 * s1);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4_t x = acc[(4 * t + i) * 256 + t256];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][4 * i + e] = scaled(o[t][4 * i + e], f0) + scaled(x[e], f1);
      }
    m = mn;
    mc = mcn;
    patch_from = min(patch_from, sh.patch_from);
  }
  const AttnArgs b = reload_args();
  // What was taken out of tiles with masks belongs to the rows that do attend to it.
  auto patch_of = [&](int d) {  // dims d .. d + 3 of this lane's row
    float4_t add = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int key = patch_from; key < min(kend, tiles * KEYS); ++key) {
      const E* v = (const E*)b.v + kv * b.v_head + d;
      if constexpr (PAGED) {
        const int p = load_const(b.table, (int64_t)seq * b.table_stride + (key >> b.log2_block));
        if ((unsigned)p >= (unsigned)b.num_pages) continue;
        v += p * b.v_page + (key & ((1 << b.log2_block) - 1)) * b.v_token;
      } else {
        v += (int64_t)(tok0 + key) * b.v_token;
      }
      if (TREE ? node.sees(sk, key) : key <= limit) add += nonfinite_of<E>(*reinterpret_cast<const u32x2*>(v));
    }
    return add;
  };
  if (part) {
    if (my_row < rows) {
      const int r = my_row - row0;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          store_global(TREE ? part + 4 * (256 * (4 * t + i) + 64 * wave + lane) : part + r * HDP + 32 * t + 8 * i + 4 * half,
                       float4_t{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]});
      int first_half = half;
      asm volatile("" : "+v"(first_half));  // compared here, not kept in scalar registers for the whole loop
      if (first_half == 0) {
        store_global(part + kFlashRows * HDP + r, m == -__builtin_inff() ? m : mc);
        store_global(part + kFlashRows * HDP + kFlashRows + r, sum);
      }
    }
    if (__builtin_expect(patch_from < kend, 0) && my_row < rows)
      for (int d = 4 * half; d < b.head_dim; d += 8)
        *reinterpret_cast<float4_t*>(TREE ? part + 4 * (256 * (d / 8) + 64 * wave + lane) : part + (my_row - row0) * HDP + d) +=
            patch_of(d);
    return;
  }
  const int group_heads = b.heads / b.kv_heads, out_row = min(my_row, rows - 1), out_tok = out_row / group_heads;
  const int out_head = kv * group_heads + (out_row - out_tok * group_heads);
  E* const out = (E*)b.out + (size_t)(tok0 + out_tok) * b.out_token + (size_t)out_head * b.out_head;
  const float inv = m == -__builtin_inff() && sum == 0.0f ? 0.0f : 1.0f / sum;  // no keys: zeros
  if (my_row < rows) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * t + 8 * i + 4 * half;
        if (d < b.head_dim)
          store_global(out + d, u32x2{Elem<E>::pack(o[t][4 * i] * inv, o[t][4 * i + 1] * inv),
                                      Elem<E>::pack(o[t][4 * i + 2] * inv, o[t][4 * i + 3] * inv)});
      }
  }
  if (__builtin_expect(patch_from < kend, 0) && my_row < rows) {
    for (int d = 4 * half; d < b.head_dim; d += 8) {
      const float4_t add = patch_of(d);
      u32x2* const at = reinterpret_cast<u32x2*>(out + d);
      const u32x2 x = *at;
      *at = u32x2{Elem<E>::pack(Elem<E>::lo(x[0]) + add[0], Elem<E>::hi(x[0]) + add[1]),
                  Elem<E>::pack(Elem<E>::lo(x[1]) + add[2], Elem<E>::hi(x[1]) + add[3])};
    }
  }
}

// Zeros in the rows of out that are in no sequence.
template <class E>
__device__ __forceinline__ void zero_rows(const AttnArgs& a, int64_t at, int64_t step) {
  const int t0 = seq_offset(a.cu, a.seqs, a.seqs, a.tokens);
  const int cpr = a.head_dim / 8, per_row = a.heads * cpr;
  for (int64_t i = at; i < (int64_t)(a.tokens - t0) * per_row; i += step) {
    const int64_t t = i / per_row;
    const int r = (int)(i - t * per_row), h = r / cpr;
    store_global((E*)a.out + (t0 + t) * a.out_token + h * a.out_head + 8 * (r - h * cpr), u32x4{0, 0, 0, 0});
  }
}

// Row tile number `rank` of all sequences' (64 at most) in the order of their last keys, the longest first: the workgroups
// that take longest then start first, whatever order the sequences come in.  The length of tile i of a sequence is (its
// cached keys x rep + 128 (i + 1)) >> q, so how many of its tiles are at least so long needs no loop: lane s counts those
// of sequence s, and a search over lengths ends at the one of tile `rank`.  False: there are only *total tiles.
template <bool PAGED>
__device__ __forceinline__ bool longest_tile(const AttnArgs& a, int rep, int min_rows, int rank, int lane, int* seq,
                                             int* tile, int* total) {
  int rows = 0;
  int64_t base = 0;
  if (lane < a.seqs) {
    const int len = max(seq_offset(a.cu, lane + 1, a.seqs, a.tokens) - seq_offset(a.cu, lane, a.seqs, a.tokens), 0);
    rows = len * rep;
    base = (int64_t)seq_keys<PAGED>(a, lane, len).before() * rep;
  }
  const int tiles = rows < min_rows ? 0 : (rows + kFlashRows - 1) / kFlashRows;
  const int q = 32 - __clz(64 * rep - 1);  // lengths in steps of 64 keys or a little more
  auto at_least = [&](int length) {        // tiles of this lane's sequence
    const int64_t above = ((int64_t)length << q) - base;
    const int64_t first = above <= 0 ? 0 : (above + kFlashRows - 1) / kFlashRows - 1;
    return tiles - (int)min(first, (int64_t)tiles);
  };
  int top = tiles ? (int)((base + (int64_t)tiles * kFlashRows) >> q) : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max(top, __shfl_xor(top, off));
  auto all = [](int v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); };
  *total = all(tiles);
  if (rank >= *total) return false;
  int lo = 0, hi = __builtin_amdgcn_readfirstlane(top) + 1;  // at least lo: more than `rank` tiles; at least hi: not
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (all(at_least(mid)) > rank) lo = mid;
    else hi = mid;
  }
  const int longer = at_least(hi), here = at_least(lo) - longer;
  const int index = rank - all(longer);  // among the tiles of this length, sequence by sequence
  const int before = wave_prefix(here) - here;
  const uint64_t mine = __ballot(index >= before && index < before + here);
  if (mine == 0) return false;
  const int owner = __builtin_amdgcn_readfirstlane(__builtin_ctzll(mine));
  *seq = owner;
  *tile = __builtin_amdgcn_readlane(tiles - at_least(lo) + index - before, owner);
  return true;
}

// One workgroup per row tile and KV head: `block` of `blocks`.
template <class E, int HDP, Keys KEYS_OF, int GROUPS>
__device__ __forceinline__ void flash_block(const AttnArgs& a, FlashShared<HDP, GROUPS>& sh, unsigned block, unsigned blocks,
                                            int rep, int min_rows, int longest_first, float scale_log2) {
  const int kv = (int)(block % a.kv_heads);
  const int numbers = (int)(blocks / a.kv_heads), number = (int)(block / a.kv_heads);
  int seq, tile, total;
  if (longest_first) {
    if (!longest_tile<KEYS_OF != Keys::kPacked>(a, rep, min_rows, number, threadIdx.x & 63, &seq, &tile, &total)) {
      if (a.zero_rest && kv == 0)
        zero_rows<E>(a, (int64_t)(number - total) * GROUPS * kFlashThreads + threadIdx.x,
                     (int64_t)(numbers - total) * GROUPS * kFlashThreads);
      return;
    }
  } else {
    // In the sequences' order, the last tiles, which have the most keys, first.
    const int t = numbers - 1 - number;
    int first;
    seq = find_seq<kFlashRows>(a.cu, a.seqs, a.tokens, rep, t, threadIdx.x & 63, &first);
    if (seq == a.seqs) {
      if (a.zero_rest && kv == 0)
        zero_rows<E>(a, (int64_t)(t - first) * GROUPS * kFlashThreads + threadIdx.x,
                     (int64_t)(numbers - first) * GROUPS * kFlashThreads);
      return;
    }
    tile = t - first;
    const int rows =
        max(seq_offset(a.cu, seq + 1, a.seqs, a.tokens) - seq_offset(a.cu, seq, a.seqs, a.tokens), 0) * rep;
    if (tile * kFlashRows >= rows || rows < min_rows) return;
  }
  const int row0 = tile * kFlashRows;
  const int tok0 = seq_offset(a.cu, seq, a.seqs, a.tokens);
  const int len = max(seq_offset(a.cu, seq + 1, a.seqs, a.tokens) - tok0, 0);
  flash_item<E, HDP, KEYS_OF, GROUPS>(a, sh, rep, scale_log2, seq, tok0, len, seq_keys<KEYS_OF != Keys::kPacked>(a, seq, len), row0,
                                      kv, 0, 0x7fffffff / FlashConfig<HDP>::KEYS, nullptr);
}

template <class E, int HDP, Keys KEYS_OF, int GROUPS>
__global__ __launch_bounds__(GROUPS * kFlashThreads, flash_waves_per_simd(HDP, GROUPS > 1)) void flash_attention_kernel(
    AttnArgs a, int rep, int min_rows, int longest_first, float scale_log2) {
  __shared__ FlashShared<HDP, GROUPS> sh;
  flash_block<E, HDP, KEYS_OF, GROUPS>(a, sh, blockIdx.x, gridDim.x, rep, min_rows, longest_first, scale_log2);
}

// A batch of both kinds of requests in one launch: the first few_grid workgroups, of which two wavefronts work, take the
// requests of at most few_rows rows (kf_few_rows.h), the others the row tiles of the rest.  The ones wait for memory
// and the others for the matrix cores, and a CU holds some of each.  24 requests of 1 .. 700 tokens over 30 .. 4000 (8 KV
// heads of 128) take 71 us, in two launches 91; 64 of 1 .. 200 over 500 .. 8000 213 (252).
template <int HDP>
using MixedFew = FewConfig<HDP, 2, 2, 2>;  // 64 dims: half the buffers, so that a CU holds four workgroups as without it
template <int HDP>
union MixedShared {
  FewShared<MixedFew<HDP>> few;
  FlashShared<HDP, 1> many;
};
template <class E, int HDP>
__global__ __launch_bounds__(kFlashThreads, flash_waves_per_simd(HDP, false)) void mixed_attention_kernel(
    AttnArgs a, int rep, int few_rows, int few_grid, int longest_first, float scale_log2, float* ws, Piece* pieces) {
  __shared__ MixedShared<HDP> sh;
  if ((int)blockIdx.x < few_grid) {  // zeros the rows behind the last request too
    if (threadIdx.x >= MixedFew<HDP>::THREADS) return;
    few_rows_stretch<E, MixedFew<HDP>, true, false>(a, sh.few, (int)blockIdx.x, few_grid, rep, few_rows, scale_log2,
                                         ws, pieces);
  } else {
    AttnArgs b = a;
    b.zero_rest = 0;
    flash_block<E, HDP, Keys::kPages, 1>(b, sh.many, blockIdx.x - few_grid, gridDim.x - few_grid, rep,
                                 few_rows + 1, longest_first, scale_log2);
  }
}

// Fewer row tiles than workgroups that the GPU holds, or tiles of very different length: the work of all is laid end to
// end and cut into equal stretches, as in kf_paged_attn.hip.  A row tile i of a sequence counts base + 2 (i + 1) steps
// of 64 / rep keys: its first row's keys and some for beginning and ending it, then the rows'.  Items are in the order
// request, KV head, row tile, and neighbouring stretches run on one XCD, whose L2 then holds their head's keys.
constexpr int kFlashItem = 128;  // keys that beginning and ending an item takes as long as
struct FlashWork {
  int rows, tiles, base, head_cost;  // head_cost: of a KV head's row tiles together
  __device__ __forceinline__ int64_t upto(int n) const { return (int64_t)n * base + (int64_t)n * (n + 1); }
};
template <bool PAGED>
__device__ __forceinline__ FlashWork flash_work(const AttnArgs& a, int s, int rep, int min_rows) {
  const int len = max(seq_offset(a.cu, s + 1, a.seqs, a.tokens) - seq_offset(a.cu, s, a.seqs, a.tokens), 0);
  FlashWork w;
  w.rows = len * rep;
  w.tiles = w.rows < min_rows ? 0 : (w.rows + kFlashRows - 1) / kFlashRows;
  w.base = (int)(((int64_t)(seq_keys<PAGED>(a, s, len).before() + kFlashItem) * rep) >> 6);
  // Never reached by offsets that ascend (flash_plan); with others no cost is above kNoWork.
  w.head_cost = (int)min(w.upto(w.tiles), (int64_t)(0x7fffffff / a.kv_heads));
  return w;
}

template <class E, int HDP, Keys KEYS_OF>
__global__ __launch_bounds__(kFlashThreads, flash_waves_per_simd(HDP, true)) void flash_cut_kernel(
    AttnArgs args) {
  constexpr bool PAGED = KEYS_OF != Keys::kPacked;
  __shared__ FlashShared<HDP, 1> sh;
  __shared__ int scan[kFlashWaves], found[2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups go to the 8 XCDs in turn: XCD x takes stretches x * grid / 8 and on.
  const int me = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  int begin, end, per;
  {
    const AttnArgs& a = args;
    const int rep = a.rep, min_rows = a.min_rows;
    if (a.zero_rest) zero_rows<E>(a, (int64_t)blockIdx.x * kFlashThreads + tid, (int64_t)gridDim.x * kFlashThreads);
    const int run = (a.seqs + kFlashThreads - 1) / kFlashThreads;
    const int s0 = min(tid * run, a.seqs), s1 = min(s0 + run, a.seqs);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine = add_work(mine, flash_work<PAGED>(a, s, rep, min_rows).head_cost * a.kv_heads);
    const int upto = work_prefix(mine);
    if (lane == 63) scan[wave] = upto;
    if (tid == 0) {
      found[0] = -1;
      static_cast<Piece*>(a.pieces)[me].seq = -1;
    }
    __syncthreads();
    int total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < kFlashWaves; ++w) {
      if (w < wave) before = add_work(before, scan[w]);
      total = add_work(total, scan[w]);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (total == kNoWork) total = 0;
    // No stretch is shorter than what a tile of keys counts.
    per = max(total / (int)gridDim.x + 1, 4 * rep + 8);
    const Stretch stretch = stretch_of(total, per, me);
    begin = stretch.begin, end = stretch.end;
    if (stretch.begins_in(before, mine)) {
      int at = before;
      for (int s = s0; s < s1; ++s) {
        const int n = flash_work<PAGED>(a, s, rep, min_rows).head_cost * a.kv_heads;
        if (begin < at + n) {
          found[0] = s;
          found[1] = at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  int seq = __builtin_amdgcn_readfirstlane(found[0]), seq_at = __builtin_amdgcn_readfirstlane(found[1]);
  if (seq < 0) return;
  begin = __builtin_amdgcn_readfirstlane(begin), end = __builtin_amdgcn_readfirstlane(end);
  per = __builtin_amdgcn_readfirstlane(per);
  for (int at = begin; at < end;) {
    const AttnArgs a = reload_args();
    const int rep = a.rep, min_rows = a.min_rows;
    FlashWork w;
    while ((w = flash_work<PAGED>(a, seq, rep, min_rows)).head_cost * a.kv_heads <= at - seq_at) {
      seq_at += w.head_cost * a.kv_heads;
      if (++seq >= a.seqs) return;
    }
    const int kv = (at - seq_at) / w.head_cost, head_at = seq_at + kv * w.head_cost, rest = at - head_at;
    // The last row tile whose predecessors count at most `rest`: n^2 + (1 + base) n <= rest.
    const double h = 0.5 * (1.0 + w.base);
    int tile = __builtin_amdgcn_readfirstlane(min(max((int)(sqrt(h * h + rest) - h), 0), w.tiles - 1));
    while (tile > 0 && w.upto(tile) > rest) --tile;
    while (tile + 1 < w.tiles && w.upto(tile + 1) <= rest) ++tile;
    tile = __builtin_amdgcn_readfirstlane(tile);
    const int item_at = head_at + (int)w.upto(tile), cost = w.base + 2 * (tile + 1);
    const int from = at - item_at, to = min(cost, end - item_at);
    const int row0 = tile * kFlashRows, len = w.rows / rep;
    const int kend = seq_keys<PAGED>(a, seq, len).last_key(min(row0 + kFlashRows - 1, w.rows - 1) / rep) + 1;
    // The part's tiles: floor(position * tiles / cost), the same for a piece's end and the next one's beginning.
    const double tiles = max((kend + FlashConfig<HDP>::KEYS - 1) / FlashConfig<HDP>::KEYS, 1), each = cost;
    const int t0 = __builtin_amdgcn_readfirstlane((int)(from * tiles / each));
    const int t1 = __builtin_amdgcn_readfirstlane((int)(to * tiles / each));
    at = item_at + cost;
    // Not begun yet.  Further on a piece has a tile, or, where a table is too narrow for its request, may have none: that
    // is written as such.
    if (t1 == 0) continue;
    const bool whole = t0 == 0 && to == cost;
    float* const part = static_cast<float*>(a.ws) + (size_t)(2 * me + (t0 == 0 ? 1 : 0)) * kFlashRows * (HDP + 2);
    if (tid == 0 && t0 == 0 && !whole) static_cast<Piece*>(a.pieces)[me] = Piece{seq, row0, kv, last_stretch(item_at, cost, per)};
    flash_item<E, HDP, KEYS_OF, 1>(a, sh, rep, a.scale_log2, seq, seq_offset(a.cu, seq, a.seqs, a.tokens), len,
                                   seq_keys<PAGED>(a, seq, len), row0, kv, t0, t1, whole ? nullptr : part);
    lds_barrier();  // the tiles have been read: the buffers are free
  }
}

// Trees of new tokens, whose row tiles all see the same keys: each (request, KV head, row tile) is cut into pieces of at most `per`
// key tiles, one a workgroup, with the smallest per for which there are workgroups enough.  So a workgroup begins once
// only, which takes as long as four or five tiles of 64 keys, and all pieces end together.  Equal stretches as above, which
// can hold the end of one item and the beginning of the next, took 59 in place of 41 us for 8 requests of 256 rows over 500
// .. 4000 keys, 37 (29) for 16 of 30 .. 186 over 100 .. 8000 (2 KV heads), both with their join; the joins 18 .. 24 (6 .. 9)
// and, of 24 items in 512 stretches, 72 (7).
//   What bounds it: long requests the bytes of K and V (two of 108 rows over up to 131071 keys, 8 KV heads of 128: 182 us,
// 5.7 TB/s, and 7 the join); others latency: 16 of 30 .. 186 rows over 100 .. 8000 keys, 24 MB, take 19.9 us, of which 2.0
// finding the piece, 2.0 until the queries and pages are there, 1.6 until the first tiles are, 2.3 two tiles of 64 keys, 3.3
// joining the groups and writing the piece; the join 5.5.
constexpr int kTreeLeast = 4;  // key tiles of a piece; with 2 and 8 the same to 1 us
struct __attribute__((aligned(16))) TreeItem {
  int tok0, row0, rows, kv;  // its request's first token, its first row, the request's rows
  int first, pieces;         // the workgroup of its first piece
};
struct TreeSpace {
  float* parts;   // [grid][kFlashRows (HDP + 2)]
  int* count;     // of items, once they are all in the list; padded to 16 bytes
  TreeItem* list;
};
template <int HDP>
__device__ __host__ inline TreeSpace tree_space(void* ws, int grid) {
  TreeSpace s;
  s.parts = static_cast<float*>(ws);
  s.count = reinterpret_cast<int*>(s.parts + (size_t)grid * kFlashRows * (HDP + 2));
  s.list = reinterpret_cast<TreeItem*>(s.count + 4);
  return s;
}
struct TreeWork {
  int tok0, rows, tiles, key_tiles;  // row tiles; tiles of keys of each
  SeqKeys sk;
};
template <int HDP>
__device__ __forceinline__ TreeWork tree_work(const AttnArgs& a, int s, int rep) {
  constexpr int KEYS = FlashConfig<HDP>::KEYS;
  TreeWork w;
  w.tok0 = seq_offset(a.cu, s, a.seqs, a.tokens);
  const int len = max(seq_offset(a.cu, s + 1, a.seqs, a.tokens) - w.tok0, 0);
  w.sk = seq_keys<true>(a, s, len);
  w.rows = len * rep;
  w.tiles = (w.rows + kFlashRows - 1) / kFlashRows;
  w.key_tiles = max((w.sk.keys + KEYS - 1) / KEYS, 1);
  return w;
}
// Sums that no lengths make wrap: at kNoWork they stay (kf_stretch.h).
__device__ __forceinline__ int times_work(int a, int b) { return (int)min((int64_t)a * b, (int64_t)kNoWork); }
__device__ __forceinline__ int all_work(int v) { return __builtin_amdgcn_readlane(work_prefix(v), 63); }

template <class E, int HDP, int GROUPS>
__global__ __launch_bounds__(GROUPS* kFlashThreads, flash_waves_per_simd(HDP, true)) void tree_cut_kernel(AttnArgs args) {
  __shared__ FlashShared<HDP, GROUPS> sh;
  __shared__ struct {
    int seq, tok0, len, keys, shift, kv, tile, piece, pieces, per, item;
  } mine;
  const int tid = threadIdx.x, lane = tid & 63;
  // Workgroups go to the 8 XCDs in turn: XCD x takes pieces x * grid / 8 and on, so that the row tiles of one KV head, which read
  // the same keys, share an L2.
  const int me = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  {
    const AttnArgs& a = args;
    const int rep = a.rep, grid = gridDim.x;
    if (tid < 64) {
      // Every lane takes a run of requests: one, as a rule.
      const int run = (a.seqs + 63) / 64, s0 = min(lane * run, a.seqs), s1 = min(s0 + run, a.seqs);
      const TreeWork none = {0, 0, 0, 1, {0, 0}}, first = s0 < s1 ? tree_work<HDP>(a, s0, rep) : none;
      auto of_run = [&](auto&& f) {  // f(request, its work) of the lane's requests
        if (s0 < s1) f(s0, first);
        for (int s = s0 + 1; s < s1; ++s) f(s, tree_work<HDP>(a, s, rep));
      };
      int items = 0, work = 0, longest = 1;
      of_run([&](int, const TreeWork& w) {
        const int n = times_work(w.tiles, a.kv_heads);
        items = add_work(items, n);
        work = add_work(work, times_work(n, w.key_tiles));
        longest = max(longest, w.key_tiles);
      });
      auto pieces_of = [&](const TreeWork& w, int per) {
        return times_work(times_work(w.tiles, a.kv_heads), (w.key_tiles + per - 1) / per);
      };
      auto all_pieces = [&](int per) {  // of this lane's requests
        int n = 0;
        of_run([&](int, const TreeWork& w) { n = add_work(n, pieces_of(w, per)); });
        return n;
      };
      const int total_items = all_work(items), total = all_work(work);
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) longest = max(longest, __shfl_xor(longest, off));
      // The smallest number of key tiles a piece, kTreeLeast or more, for which there are workgroups enough: more than
      // total / (grid + 1), at most total / (grid - items) + 1.
      int low = max(total / (grid + 1), kTreeLeast - 1);  // not enough, or fewer than that
      int high = total_items < grid ? min(total / (grid - total_items) + 1, longest) : longest;
      high = max(high, low + 1);
      while (high - low > 1) {
        const int per = low + ((high - low) >> 1);
        if (all_work(all_pieces(per)) <= grid) high = per;
        else low = per;
      }
      const int here = all_pieces(high), upto = work_prefix(here), items_upto = work_prefix(items);
      if (lane == 0) mine.seq = -1;
      int at = upto - here, item = items_upto - items;
      if (upto != kNoWork && me >= at && me < upto) {
        bool found = false;
        of_run([&](int s, const TreeWork& w) {
          const int n = pieces_of(w, high);
          if (!found && me < at + n) {
            const int pieces = (w.key_tiles + high - 1) / high;
            const int i = (me - at) / pieces;  // items in the order KV head, row tile
            mine.seq = s;
            mine.tok0 = w.tok0;
            mine.len = w.rows / rep;
            mine.keys = w.sk.keys;
            mine.shift = w.sk.shift;
            mine.kv = i / w.tiles;
            mine.tile = i - mine.kv * w.tiles;
            mine.piece = (me - at) - i * pieces;
            mine.pieces = pieces;
            mine.per = high;
            mine.item = item + i;
            found = true;
          }
          at += n;
          item += times_work(w.tiles, a.kv_heads);
        });
      }
      // Offsets that do not ascend can make more pieces than workgroups: none is joined then.
      const int all = __builtin_amdgcn_readlane(upto, 63);
      if (me == 0 && lane == 0) *tree_space<HDP>(a.ws, grid).count = all <= grid ? min(total_items, a.items) : 0;
    }
    if (a.zero_rest) zero_rows<E>(a, (int64_t)me * GROUPS * kFlashThreads + tid, (int64_t)gridDim.x * GROUPS * kFlashThreads);
    __syncthreads();
  }
  const int seq = __builtin_amdgcn_readfirstlane(mine.seq);
  if (seq < 0) return;
  const AttnArgs a = reload_args();
  const int kv = __builtin_amdgcn_readfirstlane(mine.kv), tile = __builtin_amdgcn_readfirstlane(mine.tile);
  const int piece = __builtin_amdgcn_readfirstlane(mine.piece), pieces = __builtin_amdgcn_readfirstlane(mine.pieces);
  const int per = __builtin_amdgcn_readfirstlane(mine.per), item = __builtin_amdgcn_readfirstlane(mine.item);
  const TreeSpace space = tree_space<HDP>(a.ws, gridDim.x);
  const int tok0 = __builtin_amdgcn_readfirstlane(mine.tok0), len = __builtin_amdgcn_readfirstlane(mine.len);
  const SeqKeys sk = {__builtin_amdgcn_readfirstlane(mine.keys), __builtin_amdgcn_readfirstlane(mine.shift)};
  if (tid == 0 && piece == 0 && item < a.items)
    space.list[item] = TreeItem{tok0, tile * kFlashRows, len * a.rep, kv, me, pieces};
  flash_item<E, HDP, Keys::kTree, GROUPS>(a, sh, a.rep, a.scale_log2, seq, tok0, len, sk, tile * kFlashRows, kv, piece * per,
                                          (piece + 1) * per,
                                          pieces == 1 ? nullptr : space.parts + (size_t)me * kFlashRows * (HDP + 2));
}

// Joins the pieces of item blockIdx.x in the order of the keys.
template <class E, int HDP>
__global__ __launch_bounds__(64 * kJoinWaves) void join_tree_kernel(AttnArgs a, int grid) {
  const TreeSpace space = tree_space<HDP>(a.ws, grid);
  const int count = *space.count;
  const TreeItem t = space.list[blockIdx.x];  // loaded beside the count: the list has room for every workgroup
  const int pieces = __builtin_amdgcn_readfirstlane(t.pieces);
  if ((int)blockIdx.x >= count || pieces == 1) return;
  const int rep = a.rep, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int STRIDE = kFlashRows * (HDP + 2);
  // As the lanes held them: a workgroup has eight dims of every row, a wavefront 32 rows.
  const int r = 32 * wave + (lane & 31), d = 8 * blockIdx.y + 4 * (lane >> 5);
  if (t.row0 + r >= t.rows) return;
  const float* const from = space.parts + (size_t)t.first * STRIDE;
  const int at = 4 * (256 * blockIdx.y + 64 * wave + lane);
  float top = -__builtin_inff(), l = 0.0f;
  float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
  // As in join_pieces_kernel: nothing of a piece without keys, a NaN among scores is in the sum.
  auto factor = [](float m, float high) { return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - high); };
  auto sum = [](float x, float f) { return x != x ? x : f * x; };
  constexpr int AHEAD = 16;
  for (int p0 = 0; p0 < pieces; p0 += AHEAD) {
    float m[AHEAD], s[AHEAD], high = top;
    float4_t x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      m[j] = -__builtin_inff();
      if (p0 + j >= pieces) continue;
      const float* const p = from + (size_t)(p0 + j) * STRIDE;
      m[j] = p[kFlashRows * HDP + r];
      s[j] = p[kFlashRows * HDP + kFlashRows + r];
      x[j] = *reinterpret_cast<const float4_t*>(p + at);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) high = fmaxf(high, m[j]);
    const float old = factor(top, high);
    l = sum(l, old);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = scaled(v[e], old);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (p0 + j >= pieces) continue;
      const float f = factor(m[j], high);
      l += sum(s[j], f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += scaled(x[j][e], f);
    }
    top = high;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int row = t.row0 + r, tok = row / rep, head = t.kv * rep + (row - tok * rep);
  if (d < a.head_dim)
    store_global((E*)a.out + (size_t)(t.tok0 + tok) * a.out_token + (size_t)head * a.out_head + d,
                 u32x2{Elem<E>::pack(v[0] * inv, v[1] * inv), Elem<E>::pack(v[2] * inv, v[3] * inv)});
}

template <class E, int HDP>
hipError_t launch_tree(const AttnArgs& a, const FlashPlan& p, void* ws, hipStream_t stream) {
  AttnArgs c = a;
  c.scale_log2 = a.scale * 1.44269504088896340736f, c.rep = a.heads / a.kv_heads, c.ws = ws, c.items = p.items;
  if (p.groups > 1) tree_cut_kernel<E, HDP, flash_groups(HDP)><<<p.grid, flash_groups(HDP) * kFlashThreads, 0, stream>>>(c);
  else tree_cut_kernel<E, HDP, 1><<<p.grid, kFlashThreads, 0, stream>>>(c);
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  join_tree_kernel<E, HDP><<<dim3((unsigned)p.items, HDP / 8), 64 * kJoinWaves, 0, stream>>>(c, p.grid);
  return hipGetLastError();
}

template <class E, int HDP, Keys KEYS_OF>
hipError_t launch(const AttnArgs& a, const FlashPlan& p, int min_rows, void* ws, hipStream_t stream) {
  const int rep = a.heads / a.kv_heads;
  const float scale_log2 = a.scale * 1.44269504088896340736f;
  constexpr int GROUPS = flash_groups(HDP);
  if (!p.cut) {
    if (p.groups > 1)
      flash_attention_kernel<E, HDP, KEYS_OF, GROUPS>
          <<<p.grid, GROUPS * kFlashThreads, 0, stream>>>(a, rep, min_rows, p.longest_first, scale_log2);
    else
      flash_attention_kernel<E, HDP, KEYS_OF, 1>
          <<<p.grid, kFlashThreads, 0, stream>>>(a, rep, min_rows, p.longest_first, scale_log2);
    return hipGetLastError();
  }
  if constexpr (KEYS_OF == Keys::kTree) {
    return launch_tree<E, HDP>(a, p, ws, stream);
  } else {
    float* const parts = static_cast<float*>(ws);
    Piece* const pieces = reinterpret_cast<Piece*>(parts + (size_t)2 * p.grid * kFlashRows * (HDP + 2));
    AttnArgs c = a;
    c.scale_log2 = scale_log2, c.rep = rep, c.min_rows = min_rows, c.ws = parts, c.pieces = pieces;
    flash_cut_kernel<E, HDP, KEYS_OF><<<p.grid, kFlashThreads, 0, stream>>>(c);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    join_pieces_kernel<E, HDP, kFlashRows>
        <<<join_grid<HDP, kFlashRows>(p.grid), 64 * kJoinWaves, 0, stream>>>(a, rep, parts, pieces);
    return hipGetLastError();
  }
}

template <class E, int HDP>
hipError_t launch_mixed(const AttnArgs& a, const FewPlan& f, const FlashPlan& p, int few_rows, void* ws, hipStream_t stream) {
  const int rep = a.heads / a.kv_heads;
  const float scale_log2 = a.scale * 1.44269504088896340736f;
  float* const parts = static_cast<float*>(ws);
  Piece* const pieces = reinterpret_cast<Piece*>(parts + (size_t)2 * f.grid * 32 * (HDP + 2));
  mixed_attention_kernel<E, HDP><<<f.grid + p.grid, kFlashThreads, 0, stream>>>(a, rep, few_rows, f.grid, p.longest_first,
                                                                                scale_log2, parts, pieces);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  join_pieces_kernel<E, HDP, 32><<<join_grid<HDP, 32>(f.grid), 64 * kJoinWaves, 0, stream>>>(a, rep, parts, pieces);
  return hipGetLastError();
}

template <class E, Keys KEYS_OF>
hipError_t launch_dim(const AttnArgs& a, const FlashPlan& p, int min_rows, void* ws, hipStream_t stream) {
  if (a.head_dim <= 64) return launch<E, 64, KEYS_OF>(a, p, min_rows, ws, stream);
  if (a.head_dim <= 128) return launch<E, 128, KEYS_OF>(a, p, min_rows, ws, stream);
  return launch<E, 256, KEYS_OF>(a, p, min_rows, ws, stream);
}

}  // namespace

// How the row tiles are spread, by their number (`items`, from above) and the longest a sequence can be (`keys`: over a
// cache the table's width, as lengths are on the device; a first chunk of 2000 tokens, 12 heads on 2 of 128, takes 39 us
// with a table of its length and, cut, 56 with one of 131072 tokens).  The
// kernel's time is at least its longest item's, so where there are few and they are long they are
//   cut         into equal stretches that a second launch joins, where the CUs that would stay idle make up for writing and
//               reading the pieces: 200 tokens over 60000 (8 KV heads of 128, 56 items) 1392 -> 285 us; but 2000 tokens of
//               12 heads 35 -> 64, 16 ragged prompts 49 -> 79, a mixed batch 91 -> 102 us;
//   shared      by two groups of four wavefronts, where a CU gets hardly more than half the workgroups it could hold (four of
//               up to 64 dims, two of 128): 2000 tokens of 12 heads of 128 (192 items) 45 -> 35 us, 4000 of 8 of 96 (250)
//               91 -> 70, 2047 tokens of 32 of 64 over 29999 (512) 666 -> 613, 1600 (400) 27.9 -> 24.4; but 16 ragged prompts
//               of 128 dims (700) 49 -> 65, as eight wavefronts at one barrier overlap less than two workgroups do;
//   longest first, where they do not all run at once: 16 ragged prompts 57 -> 49 us, a mixed batch 105 -> 91.
FlashPlan flash_plan(const AttnArgs& a, bool paged, int cu_count) {
  FlashPlan p;
  const int64_t rep = a.heads / a.kv_heads;
  const int64_t tiles = a.tokens * rep / kFlashRows + a.seqs + 1;
  const int hdp = a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256;
  const int64_t keys = paged ? (int64_t)a.table_width << a.log2_block : a.tokens;
  const int64_t most_cost = (tiles + a.seqs) * a.kv_heads * (((keys + kFlashItem) * rep >> 6) + 2 * tiles + 2);
  const int64_t items = tiles * a.kv_heads;
  p.cut = items < cu_count && keys * (cu_count - items) > (int64_t)1600 * cu_count && most_cost < kNoWork;
  p.groups = (hdp == 64 ? 2 : 4) * items <= 5 * cu_count && keys > 256 ? flash_groups(hdp) : 1;
  // One sequence has its longest tiles last in any case, and workgroups that all run at once need no order.
  p.longest_first = a.seqs > 1 && a.seqs <= 64 && items * p.groups > cu_count * flash_waves_per_simd(hdp, false);
  p.grid = p.cut ? cu_count * flash_waves_per_simd(hdp, true) : (int)items;
  p.items = 0;
  return p;
}

// For trees (us over 8 KV heads of 128 as a rule):
//   cut         as above, into pieces, where there are as many workgroups as items and more than 768 keys: below, the second
//               launch costs more than the pieces spare (8 requests of 128 rows over 200 .. 500 keys 18 / 24 cut, 400 .. 700
//               22 / 25; 64 rows over 1000 keys 22 / 18).  8 of 256 rows over 500 .. 4000 57 / 37, 16 of 30 .. 150 over 100 ..
//               8000 (2 KV heads) 91 / 26, 24 of 96 over 500 .. 4000 61 / 49, 2 of 108 over up to 131071 1880 / 196.
//   two groups  of wavefronts a workgroup where there are two or more pieces an item: half as many pieces to write and join (2 of
//               108 rows over up to 131071 keys 200 / 196, 4 of 80 over 40000 118 / 116, one of 320 over 30000, 64 dims, 37 / 32).
//               With more items two workgroups a CU even them out better (three of up to 64 dims): 128 of 12 rows over 4000 keys
//               (2 KV heads) 74 two groups / 41 two workgroups, 64 of 100 .. 190 rows of 64 dims 44 / 38.
FlashPlan tree_plan(const AttnArgs& a, int cu_count) {
  FlashPlan p = flash_plan(a, true, cu_count);
  const int64_t rep = a.heads / a.kv_heads, keys = (int64_t)a.table_width << a.log2_block;
  const int64_t items = (a.tokens * rep / kFlashRows + a.seqs + 1) * a.kv_heads;
  const int hdp = a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256;
  const int held = flash_waves_per_simd(hdp, true);  // workgroups of one group that a CU holds
  const int64_t most_work = items * (keys / (hdp == 256 ? 32 : 64) + 1);
  p.cut = keys > 768 && items <= (int64_t)held * cu_count && most_work < kNoWork;
  if (!p.cut) {
    p.grid = (int)items;
    return p;
  }
  p.groups = 2 * items <= cu_count ? flash_groups(hdp) : 1;
  p.grid = (p.groups > 1 ? 1 : held) * cu_count;
  p.grid -= p.grid % 8;  // as many on every XCD
  p.items = (int)items;
  p.cut = p.grid >= items;
  if (!p.cut) p.grid = (int)items;
  return p;
}

size_t flash_workspace_bytes(int head_dim, const FlashPlan& p) {
  if (!p.cut) return 0;
  const int padded = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  if (p.items)
    return (size_t)p.grid * sizeof(float) * kFlashRows * (padded + 2) + 4 * sizeof(int) + (size_t)p.items * sizeof(TreeItem);
  return (size_t)p.grid * (2 * sizeof(float) * kFlashRows * (padded + 2) + sizeof(Piece));
}

hipError_t flash_attention_launch(const AttnArgs& a, bool paged, bool bf16, const FlashPlan& p, int min_rows, void* ws,
                                  hipStream_t stream) {
  if (a.ancestors)
    return bf16 ? launch_dim<bhalf_t, Keys::kTree>(a, p, min_rows, ws, stream)
                : launch_dim<half_t, Keys::kTree>(a, p, min_rows, ws, stream);
  if (paged)
    return bf16 ? launch_dim<bhalf_t, Keys::kPages>(a, p, min_rows, ws, stream)
                : launch_dim<half_t, Keys::kPages>(a, p, min_rows, ws, stream);
  return bf16 ? launch_dim<bhalf_t, Keys::kPacked>(a, p, min_rows, ws, stream)
              : launch_dim<half_t, Keys::kPacked>(a, p, min_rows, ws, stream);
}

hipError_t mixed_attention_launch(const AttnArgs& a, bool bf16, const FewPlan& f, const FlashPlan& p, int few_rows, void* ws,
                                  hipStream_t stream) {
  if (a.head_dim <= 64)
    return bf16 ? launch_mixed<bhalf_t, 64>(a, f, p, few_rows, ws, stream)
                : launch_mixed<half_t, 64>(a, f, p, few_rows, ws, stream);
  return bf16 ? launch_mixed<bhalf_t, 128>(a, f, p, few_rows, ws, stream)
              : launch_mixed<half_t, 128>(a, f, p, few_rows, ws, stream);
}

}  // namespace kf
