// Causal attention of packed sequences with many rows per sequence, over contiguous keys (whole prompts) or over
// the pages of a cache (chunks of prompts): one pass over the keys with the running maximum and sum of the softmax.
//
//   out[t, h] = sum_s softmax_s(scale q[t, h] . k[s, kv]) v[s, kv],   s <= position of t,   kv = h / rep
//
// A workgroup owns 128 rows of one KV head (kf_attn_tiles.h), 32 per wavefront, and walks their keys 64 at a
// time (32 for heads of more than 128, whose outputs fill half the registers) through two LDS buffers.  Scores, maximum, sum and outputs are held in 32 bits; probabilities are rounded to
// the inputs' type for the second matrix product (half a step of that type, as inputs are), the outputs once
// more when they are stored.  The maximum that the exponentials are taken against follows the true one only when it is
// exceeded by a factor 2^8: outputs and sums are then rescaled, which most tiles after the first spare.
#include "kf_attn_tiles.h"
#include "kf_launch.h"

namespace kf {
namespace {

constexpr int kFlashWaves = 4, kFlashThreads = 64 * kFlashWaves;
constexpr int kFlashRows = 32 * kFlashWaves;

// Wavefronts per SIMD that the registers have to allow: one computes scores while another works on its
// softmax.  From two on the products also accumulate in ordinary registers, without moves.
constexpr int flash_waves_per_simd(int hdp) { return hdp == 64 ? 4 : hdp == 128 ? 2 : 1; }

template <class E, int HDP, bool PAGED>
__global__ __launch_bounds__(kFlashThreads, flash_waves_per_simd(HDP)) void flash_attention_kernel(AttnArgs a, int rep, int min_rows,
                                                                        float scale_log2) {
  constexpr int ROW = HDP * 2;                      // bytes
  constexpr int KEYS = HDP == 256 ? 32 : 64, KU = KEYS / 32, KK = KEYS / 16;
  constexpr int MINE = KEYS / kFlashWaves;           // keys of a tile that a wavefront fetches
  constexpr int TILE = KEYS * ROW;
  constexpr int ST = HDP / 16;                      // k steps of the first product
  constexpr int DT = HDP / 32;                      // 32-row tiles of O^T
  // Queries of more than 128 dims leave no registers for themselves beside the outputs: each lane's stay in LDS.
  constexpr bool Q_LDS = HDP == 256;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * TILE + (Q_LDS ? kFlashRows * ROW : 0)];
  __shared__ int found[2][kFlashWaves];  // infinities or NaN in a masked tile
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = blockIdx.x % a.kv_heads;
  // The last tiles of a sequence have the most keys: they start first.
  const int tile = (int)(gridDim.x / a.kv_heads) - 1 - (int)(blockIdx.x / a.kv_heads);

  int first;
  const int seq = find_seq<kFlashRows>(a.cu, a.seqs, a.tokens, rep, tile, lane, &first);
  const int tok0 = seq_offset(a.cu, seq, a.seqs, a.tokens);
  const int len = max(seq_offset(a.cu, seq + 1, a.seqs, a.tokens) - tok0, 0);
  const int rows = len * rep;
  const int row0 = (tile - first) * kFlashRows;
  if (row0 >= rows || (seq < a.seqs && rows < min_rows)) return;

  // This lane's row.  Rows past the end repeat the last one and are not stored.
  const int my_row = row0 + 32 * wave + (lane & 31);
  const int row = min(my_row, rows - 1);
  const int tok = row / rep;
  const int head = kv * rep + (row - tok * rep);
  E* const out = (E*)a.out + (size_t)(tok0 + tok) * a.out_token + (size_t)head * a.out_head;
  if (seq == a.seqs) {
    if (a.zero_rest && my_row < rows)
      for (int c = half; c < a.head_dim / 8; c += 2) *(u32x4*)(out + 8 * c) = u32x4{0, 0, 0, 0};
    return;
  }

  // Keys: positions before this lane's row's own, itself included.
  const int seq_len = PAGED ? min(max(load_const(a.seq_lens, seq), 0), a.table_width << a.log2_block) : len;
  const int shift = seq_len - len;
  const int limit = shift + tok;  // may be negative: no keys
  const int wave_row = row0 + 32 * wave;
  const int wave_lo = shift + min(wave_row, rows - 1) / rep, wave_hi = shift + min(wave_row + 31, rows - 1) / rep;
  const int first_limit = shift + row0 / rep;  // the workgroup's first row's
  const int kend = shift + min(row0 + kFlashRows - 1, rows - 1) / rep + 1;
  const int tiles = kend <= 0 ? 0 : (kend + KEYS - 1) / KEYS;

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
  const int64_t table_at = (int64_t)seq * a.table_stride;
  auto page_of = [&](int key) {  // uniform; -1: not in the cache
    const int p = load_const(a.table, table_at + (min(key, kend - 1) >> a.log2_block));
    return (unsigned)p < (unsigned)a.num_pages ? p : -1;
  };
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
  int page = 0;
  if (tiles > 0) {
    if constexpr (PAGED) page = page_of(MINE * wave);
    issue(0, 0, page);
    if constexpr (PAGED) page = page_of(min(KEYS, kend - 1) + MINE * wave);
  }
  for (int kt = 0; kt < tiles; ++kt) {
    const uint32_t buf = (kt & 1) * 2 * TILE;
    dma_barrier();
    if (kt + 1 < tiles) {
      issue(kt + 1, 2 * TILE - buf, page);
      if constexpr (PAGED) page = page_of((kt + 2) * KEYS + MINE * wave);
    }
    const int key0 = kt * KEYS;

    // Masks: keys past a row's own, pages that are not there.
    uint32_t bad = 0;  // bit i: keys key0 + 16 i .. + 15 are not there
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < KK; ++i) bad |= page_of(key0 + 16 * i) < 0 ? 1u << i : 0u;
    }
    const uint32_t my_v = lds + buf + TILE + (uint32_t)(MINE * wave) * ROW;  // the rows of V that this wavefront looks after
    bool nonfinite = false;
    if (__builtin_expect(key0 + KEYS - 1 > first_limit || bad != 0, 0)) {  // the same in all wavefronts
      const bool any = lds_any_nonfinite<E>(my_v, MINE * ROW / 1024, lane);
      if (lane == 0) found[kt & 1][wave] = any;
      lds_barrier();
#pragma unroll
      for (int w = 0; w < kFlashWaves; ++w) nonfinite |= found[kt & 1][w] != 0;
      nonfinite = __builtin_amdgcn_readfirstlane(nonfinite);
    }
    if (__builtin_expect(nonfinite, 0)) {
      lds_finite_only<E>(my_v, MINE * ROW / 1024, lane);
      lds_barrier();
      patch_from = min(patch_from, key0);
    }
    if (key0 > wave_hi) continue;  // only other wavefronts have keys here

    float16_t s[KU];
    const uint32_t kb = lds + buf + k_at;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int u = 0; u < KU; ++u)
        s[u] = Elem<E>::mfma32(lds_read16((kb ^ (uint32_t)(32 * st)) + u * 32 * ROW), Q_LDS ? q_lds[64 * st] : qf[Q_LDS ? 0 : st], s[u]);

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
#pragma unroll
      for (int q = 0; q < 2 * KK; ++q) {
        const int last = keys_at(q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e > last) s[q >> 2][4 * (q & 3) + e] = -__builtin_inff();
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
  const float inv = m == -__builtin_inff() && sum == 0.0f ? 0.0f : 1.0f / sum;  // no keys: zeros
  if (my_row < rows) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * t + 8 * i + 4 * half;
        if (d < a.head_dim)
          *(u32x2*)(out + d) = u32x2{Elem<E>::pack(o[t][4 * i] * inv, o[t][4 * i + 1] * inv),
                                     Elem<E>::pack(o[t][4 * i + 2] * inv, o[t][4 * i + 3] * inv)};
      }
  }

  // What was taken out of tiles with masks belongs to the rows that do attend to it.
  if (__builtin_expect(patch_from < kend, 0) && my_row < rows) {
    for (int c = half; c < a.head_dim / 4; c += 2) {
      float4_t add = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int key = patch_from; key < kend; ++key) {
        const E* v = (const E*)a.v + kv * a.v_head + 4 * c;
        if constexpr (PAGED) {
          const int p = page_of(key);
          if (p < 0) continue;
          v += p * a.v_page + (key & ((1 << a.log2_block) - 1)) * a.v_token;
        } else {
          v += (int64_t)(tok0 + key) * a.v_token;
        }
        if (key <= limit) add += nonfinite_of<E>(*reinterpret_cast<const u32x2*>(v));
      }
      u32x2* const at = reinterpret_cast<u32x2*>(out + 4 * c);
      const u32x2 x = *at;
      *at = u32x2{Elem<E>::pack(Elem<E>::lo(x[0]) + add[0], Elem<E>::hi(x[0]) + add[1]),
                  Elem<E>::pack(Elem<E>::lo(x[1]) + add[2], Elem<E>::hi(x[1]) + add[3])};
    }
  }
}

template <class E, int HDP>
hipError_t launch(const AttnArgs& a, bool paged, int min_rows, hipStream_t stream) {
  const int rep = a.heads / a.kv_heads;
  const unsigned tiles = (unsigned)((int64_t)a.tokens * rep / kFlashRows + a.seqs + 1);
  const dim3 grid(tiles * (unsigned)a.kv_heads);
  const float scale_log2 = a.scale * 1.44269504088896340736f;
  if (paged) flash_attention_kernel<E, HDP, true><<<grid, kFlashThreads, 0, stream>>>(a, rep, min_rows, scale_log2);
  else flash_attention_kernel<E, HDP, false><<<grid, kFlashThreads, 0, stream>>>(a, rep, min_rows, scale_log2);
  return hipGetLastError();
}

template <class E>
hipError_t launch_dim(const AttnArgs& a, bool paged, int min_rows, hipStream_t stream) {
  if (a.head_dim <= 64) return launch<E, 64>(a, paged, min_rows, stream);
  if (a.head_dim <= 128) return launch<E, 128>(a, paged, min_rows, stream);
  return launch<E, 256>(a, paged, min_rows, stream);
}

}  // namespace

hipError_t flash_attention_launch(const AttnArgs& a, bool paged, bool bf16, int min_rows, hipStream_t stream) {
  return bf16 ? launch_dim<bhalf_t>(a, paged, min_rows, stream) : launch_dim<half_t>(a, paged, min_rows, stream);
}

}  // namespace kf
