// Pieces shared by the kernels of prompt_attention and paged_attention (kf_flash.hip, kf_paged_attn.hip):
// element types, the rows a workgroup owns, tiles of K and V in LDS and the products on them.
//
// Rows.  A row is (token, query head of the KV head's group), tokens first: row r of a sequence is its token
// r / rep with query head kv * rep + r % rep.  So the rep heads that read the same keys share every tile
// of K and V, and a single token of a grouped model already fills rep rows of a matrix instruction.
//
// Products.  Scores are computed transposed, S^T = K Q^T, so a lane holds scores of one query only (column
// lane % 32) and its maximum, its sum and the factor that rescales its outputs are plain per-lane values.
// The lane's eight scores 8 i .. 8 i + 7 of a 32-key tile are keys 16 kk + {4 h + 0..3, 8 + 4 h + 0..3} (h =
// lane / 32), which serve as they are as the right operand of O^T += V^T P^T if V^T is read with its keys
// in that order: probabilities go from one product to the next without leaving their registers.  V^T comes from
// the row-major tile of V by transposing LDS reads (ds_read_b64_tr_b16: each 16 lanes read a 4 x 16 block
// of 16-bit values, lane i of them gets column i).
#pragma once

#include "kf_device.h"
#include "kf_stretch.h"

namespace kf {

typedef __bf16 bhalf_t;
typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));

template <class E>
struct Elem;
template <>
struct Elem<half_t> {
  static constexpr uint32_t kExp = 0x7C007C00u, kExpLow = 0x04000400u;
  static __device__ __forceinline__ float16_t mfma32(u32x4 a, u32x4 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(a), bit_cast<half8_t>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4_t mfma16(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<half8_t>(a), bit_cast<half8_t>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {  // both rounded to nearest even
    const half2_t v = {(half_t)a, (half_t)b};
    return bit_cast<uint32_t>(v);
  }
  static __device__ __forceinline__ float lo(uint32_t v) { return (float)bit_cast<half2_t>(v)[0]; }
  static __device__ __forceinline__ float hi(uint32_t v) { return (float)bit_cast<half2_t>(v)[1]; }
};
template <>
struct Elem<bhalf_t> {
  static constexpr uint32_t kExp = 0x7F807F80u, kExpLow = 0x00800080u;
  static __device__ __forceinline__ float16_t mfma32(u32x4 a, u32x4 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bit_cast<bhalf8_t>(a), bit_cast<bhalf8_t>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4_t mfma16(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bit_cast<bhalf8_t>(a), bit_cast<bhalf8_t>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const bhalf2_t v = {(bhalf_t)a, (bhalf_t)b};
    return bit_cast<uint32_t>(v);
  }
  static __device__ __forceinline__ float lo(uint32_t v) { return bit_cast<float>(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return bit_cast<float>(v & 0xFFFF0000u); }
};

// Source of the 16 bytes that stand for what is not there: head sizes below the tile's, keys past the end,
// pages that are not in the cache.  Zeros keep such places finite, so a product with a zero is zero.
static __device__ __attribute__((aligned(16))) uint32_t g_attn_zeros[4] = {0, 0, 0, 0};

__device__ __forceinline__ void lds_dma16(uint32_t lds, const void* src) {
  asm volatile("global_load_lds_dwordx4 %1, off" ::"{m0}"(lds), "v"(src) : "memory");
}
// ONCE: no other workgroup reads these bytes.
template <bool ONCE>
__device__ __forceinline__ void lds_dma16(uint32_t lds, const void* base, uint32_t offset) {
  if constexpr (ONCE) asm volatile("global_load_lds_dwordx4 %1, %2 nt" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
  else asm volatile("global_load_lds_dwordx4 %1, %2" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
}
// All of this wavefront's copies have landed and its reads are done, and every wavefront of the workgroup has come
// here.
__device__ __forceinline__ void dma_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The same for LDS alone: copies go on.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The loads into v end here.  Without it the compiler waits for them where v is used, in the loop, by waiting for all
// vector memory operations: the copies of the next tile, of which it does not know, among them.
template <int N>
__device__ __forceinline__ void arrived(u32x4 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

// The 16-byte pieces of a row of a tile are stored at piece ^ swizzle(row), so that the 16 (K) or 4 (V) rows which
// one read touches lie in different banks.  (Measured: none of the kernel of many rows' LDS cycles are conflicts.)
template <int HDP>
__device__ __forceinline__ constexpr int swizzle_k(int key) {
  return HDP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int HDP>
__device__ __forceinline__ constexpr int swizzle_v(int key) {
  return HDP == 64 ? 4 * ((key >> 1) & 1) : 4 * (key & 3);
}

// V's swizzle for 16-column reads (16 x 16 products): eight rows of one read in different banks.
template <int HDP>
__device__ __forceinline__ constexpr int swizzle_v16(int key) {
  return HDP == 64 ? 2 * ((key >> 1) & 3) : 2 * (key & 7);
}

// Copies ROWS keys of K and of V into tiles, swizzled.  The source offsets of a lane do not change, so a copy of keys
// that are all there is one instruction per KiB.
// FEW: for the kernel of few rows, whose products are 16 x 16 and whose keys no other workgroup reads.
template <class E, int HDP, bool FEW, int ROWS = 16>
struct TileCopy {
  static constexpr int CPR = HDP / 8;    // 16-byte pieces per row
  static constexpr int RPI = 64 / CPR;   // rows per copy instruction
  static constexpr int N = ROWS / RPI;   // instructions per tile
  uint32_t vo_k[N], vo_v[N];
  int pieces;  // of a row that are there
  int row0;    // the first key's row in the tile, mod 16 (ROWS < 16 only)

  __device__ __forceinline__ int piece_k(int j, int lane) const {
    return (lane % CPR) ^ swizzle_k<HDP>(row0 + RPI * j + lane / CPR);
  }
  __device__ __forceinline__ int piece_v(int j, int lane) const {
    const int r = row0 + RPI * j + lane / CPR;
    return (lane % CPR) ^ (FEW ? swizzle_v16<HDP>(r) : swizzle_v<HDP>(r));
  }
  // Strides of at most 2^26 elements (checked by the caller), so offsets fit 32 bits.
  __device__ __forceinline__ TileCopy(int64_t k_token, int64_t v_token, int head_dim, int lane, int tile_row = 0)
      : pieces(head_dim / 8), row0(ROWS < 16 ? tile_row & 15 : 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t r = RPI * j + lane / CPR;
      vo_k[j] = 2u * (r * (uint32_t)k_token + 8u * piece_k(j, lane));
      vo_v[j] = 2u * (r * (uint32_t)v_token + 8u * piece_v(j, lane));
    }
  }
  // kb, vb: the first key's values; `rows` of the keys are there (any value), the others and the pieces past
  // the head size become zeros.
  __device__ __forceinline__ void operator()(uint32_t dst_k, uint32_t dst_v, const E* kb, const E* vb, int rows,
                                             int lane) const {
    if (rows >= ROWS && pieces == CPR) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        lds_dma16<FEW>(dst_k + 1024 * j, kb, vo_k[j]);
        lds_dma16<FEW>(dst_v + 1024 * j, vb, vo_v[j]);
      }
      return;
    }
    int there = pieces, lane_here = lane;
    // The comparisons below are made here, not kept in registers for the whole loop.
    asm volatile("" : "+s"(there), "+v"(lane_here));
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bool row_ok = RPI * j + lane_here / CPR < rows;
      uint32_t ok = vo_k[j], ov = vo_v[j];
      asm volatile("" : "+v"(ok), "+v"(ov));  // nor are offsets as 64 bits
      const char* const sk = reinterpret_cast<const char*>(kb) + ok;
      const char* const sv = reinterpret_cast<const char*>(vb) + ov;
      lds_dma16(dst_k + 1024 * j, row_ok && piece_k(j, lane_here) < there ? sk : (const char*)g_attn_zeros);
      lds_dma16(dst_v + 1024 * j, row_ok && piece_v(j, lane_here) < there ? sv : (const char*)g_attn_zeros);
    }
  }
};

// 4 x 16 transposing read of 16-bit values: see the head of this file.
__device__ __forceinline__ u32x2 lds_read_tr(uint32_t lds) {
  typedef __attribute__((address_space(3))) short4_t* ptr_t;
  return bit_cast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr_t)(uintptr_t)lds));
}
__device__ __forceinline__ u32x4 lds_read16(uint32_t lds) {
  typedef const __attribute__((address_space(3))) u32x4* ptr_t;
  return *(ptr_t)(uintptr_t)lds;
}

__device__ __forceinline__ u32x2 lds_read8(uint32_t lds) {
  typedef const __attribute__((address_space(3))) u32x2* ptr_t;
  return *(ptr_t)(uintptr_t)lds;
}

__device__ __forceinline__ float max_halves(float v) {  // of lanes l and l ^ 32
  const auto s = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return fmaxf(bit_cast<float>((uint32_t)s[0]), bit_cast<float>((uint32_t)s[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return bit_cast<float>((uint32_t)s[0]) + bit_cast<float>((uint32_t)s[1]);
}

// Whether any 16-bit value of the four words is infinite or NaN.
template <class E>
__device__ __forceinline__ bool any_nonfinite(u32x4 v) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) t |= (v[i] & Elem<E>::kExp) + Elem<E>::kExpLow;
  return (t & 0x80008000u) != 0;
}

// V next to masked keys.  A masked key may hold infinities or NaN, which a probability of zero does not cancel.  So
// where a tile has both, the values that are not finite become zeros in LDS before its product, and are added to the
// outputs of the rows that attend to their keys one key after the other.
template <class E>
__device__ __forceinline__ u32x4 finite_only(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t inf = Elem<E>::kExp;
    if ((v[i] & inf & 0xFFFFu) == (inf & 0xFFFFu)) v[i] &= 0xFFFF0000u;
    if ((v[i] & inf & 0xFFFF0000u) == (inf & 0xFFFF0000u)) v[i] &= 0x0000FFFFu;
  }
  return v;
}
// ... of `kib` KiB of a tile from lds on, read and written by one wavefront.
template <class E>
__device__ __forceinline__ bool lds_any_nonfinite(uint32_t lds, int kib, int lane) {
  bool any = false;
  for (int i = 0; i < kib; ++i) any |= any_nonfinite<E>(lds_read16(lds + 1024 * i + 16 * lane));
  return __ballot(any) != 0;
}
template <class E>
__device__ __forceinline__ void lds_finite_only(uint32_t lds, int kib, int lane) {
  typedef __attribute__((address_space(3))) u32x4* ptr_t;
#pragma unroll 1
  for (int i = 0; i < kib; ++i) {
    const uint32_t at = lds + 1024 * i + 16 * lane;
    *(ptr_t)(uintptr_t)at = finite_only<E>(lds_read16(at));
  }
}
// Four values of a row of V with zeros for the finite ones.
template <class E>
__device__ __forceinline__ float4_t nonfinite_of(u32x2 v) {
  const float4_t x = {Elem<E>::lo(v[0]), Elem<E>::hi(v[0]), Elem<E>::lo(v[1]), Elem<E>::hi(v[1])};
  float4_t y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = fabsf(x[e]) < __builtin_inff() ? 0.0f : x[e];
  return y;
}

// Lengths, offsets and pages do not change while a kernel runs: scalar loads where the index is uniform.
__device__ __forceinline__ int load_const(const int* p, int64_t i) {
  return ((const __attribute__((address_space(4))) int*)p)[i];
}
// 16 bytes of q and stores to out, as global memory (pointers read from memory would be generic ones).
__device__ __forceinline__ u32x4 load_global16(const void* p) {
  return *(const __attribute__((address_space(1))) u32x4*)p;
}
template <class V>
__device__ __forceinline__ void store_global(void* p, V v) {
  *(__attribute__((address_space(1))) V*)p = v;
}

// The kernel's first argument, read anew: what is made from it inside a loop over items is loaded there by scalar loads
// instead of being held in scalar registers, which are too few, for the whole kernel.
__device__ __forceinline__ AttnArgs reload_args() {
  typedef const __attribute__((address_space(4))) uint64_t* words_t;
  words_t p = (words_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  static_assert(sizeof(AttnArgs) % 8 == 0, "whole words");
  struct Words {
    uint64_t w[sizeof(AttnArgs) / 8];
  } v;
#pragma unroll
  for (size_t i = 0; i < sizeof(AttnArgs) / 8; ++i) v.w[i] = p[i];
  return bit_cast<AttnArgs>(v);
}

// Inclusive prefix sums over a wavefront.
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// The same of work (kf_stretch.h).
__device__ __forceinline__ int work_prefix(int v) {
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = add_work(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return v;
}

// Sequences of packed tokens: [offset(s), offset(s + 1)) for s < seqs, then the rows in no sequence as sequence
// `seqs`.  Offsets outside [0, tokens] are clamped, so no row index made from them leaves the tensors.
__device__ __forceinline__ int seq_offset(const int* cu, int s, int seqs, int tokens) {
  return s <= 0 ? 0 : s > seqs ? tokens : min(max(load_const(cu, s), 0), tokens);
}

// The keys of sequence s whose last `len` tokens are new: `keys` of them have a place in its table, and the new token t is at
// position shift + t, which may be behind them (a table that is too narrow: it attends to what has a place) or negative
// (fewer keys than new tokens: none).
struct SeqKeys {
  int keys, shift;
  __device__ __forceinline__ int last_key(int t) const { return min(shift + t, keys - 1); }  // that token t attends to
  __device__ __forceinline__ int before() const { return min(max(shift, 0), keys); }         // of the keys, not new ones
};
template <bool PAGED>
__device__ __forceinline__ SeqKeys seq_keys(const AttnArgs& a, int s, int len) {
  const int n = PAGED ? max(load_const(a.seq_lens, s), 0) : len;
  return SeqKeys{PAGED ? min(n, a.table_width << a.log2_block) : n, n - len};
}

// The keys that a node of a tree of new tokens attends to: all that were there before them, and of the new ones, of which node j
// is at key shift + j, those whose bit is set (64 at most).  Only tiles with new tokens' keys, the last of a request, ask.
struct TreeRow {
  uint64_t bits;
  __device__ __forceinline__ bool sees(const SeqKeys& sk, int key) const {
    const int node = key - sk.shift;
    return key < sk.keys && (node < 0 || (node < 64 && (bits >> node & 1)));
  }
  // Bit e: key + e, of a key that is the same in all lanes; so are the shifts.
  __device__ __forceinline__ uint64_t from(const SeqKeys& sk, int key) const {
    const int node = key - sk.shift, there = sk.keys - key;
    const uint64_t mine = node >= 64 || node <= -64 ? 0 : node >= 0 ? bits >> node : bits << -node;
    const uint64_t old = node >= 0 ? 0 : node <= -64 ? ~0ull : (1ull << -node) - 1;
    const uint64_t in = there >= 64 ? ~0ull : there <= 0 ? 0 : (1ull << there) - 1;
    return (mine | old) & in;
  }
};

// Tiles of BM rows over the packed sequences, numbered so that a tile finds its sequence without a scan: sequence
// s owns the numbers from offset(s) * rep / BM + s on, enough for its rows, as
// floor(a + b) + 1 >= floor(a) + ceil(b).  Returns the largest s <= seqs whose first number is at most t.
// 64 probes a round; all lanes return the same.
template <int BM>
__device__ __forceinline__ int find_seq(const int* cu, int seqs, int tokens, int rep, int t, int lane,
                                        int* first) {
  int lo = 0, range = seqs + 1;
  while (range > 1) {
    const int step = (range + 63) >> 6;
    const int s = lo + lane * step;
    const bool in = lane * step < range;
    const bool at_or_before = in && (lane == 0 || seq_offset(cu, s, seqs, tokens) * rep / BM + s <= t);
    // The last probe that holds: offsets that do not ascend still give a first number of at most t.
    const int n = 63 - __clzll((long long)__ballot(at_or_before));
    lo += n * step;
    range = min(step, range - n * step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  *first = lo == 0 ? 0 : seq_offset(cu, lo, seqs, tokens) * rep / BM + lo;
  return lo;
}

// What the second launch needs to know of a cut item, left by the workgroup in whose stretch it begins.
struct Piece {
  int seq, row0, kv, last;  // last: the workgroup in whose stretch it ends; seq < 0: nothing begins and goes on here
};

// A piece's output against the maximum of them all.  A factor of zero leaves nothing of it but infinities and NaN.
__device__ __forceinline__ float scaled(float x, float f) { return fabsf(x) < __builtin_inff() ? f * x : x; }

namespace {
// Joins the pieces of the items that workgroup blockIdx.x of the first launch began and did not end.  A long item can
// have hundreds, which is what takes the time: the wavefronts of a workgroup take every kJoinWaves-th piece of the
// same 64 x 4 values, kJoinAhead of them loaded at once, and the workgroups in y share an item's values, 32 at most:
// 8 requests of 1 .. 12 tokens over up to 32000 (2 KV heads of 128) take 79 us in all, with 16 workgroups 87, with 8
// 107; 64 single tokens 25.4 either way.
constexpr int kJoinWaves = 4, kJoinAhead = 8;
template <int HDP, int ROWS>
dim3 join_grid(int stretches) { return dim3(stretches, ROWS * HDP / 256 < 32 ? ROWS * HDP / 256 : 32); }

template <class E, int HDP, int ROWS>
__global__ __launch_bounds__(64 * kJoinWaves) void join_pieces_kernel(AttnArgs a, int rep, const float* ws, const Piece* pieces) {
  __shared__ float stat[2][kJoinWaves][64];
  __shared__ float4_t parts[kJoinWaves][64];
  const Piece pc = pieces[blockIdx.x];
  if (pc.seq < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tok0 = seq_offset(a.cu, pc.seq, a.seqs, a.tokens);
  const int rows = (seq_offset(a.cu, pc.seq + 1, a.seqs, a.tokens) - tok0) * rep;
  const int live_rows = min(rows - pc.row0, ROWS);
  constexpr int STRIDE = ROWS * (HDP + 2);
  const int first = blockIdx.x;
  for (int i0 = blockIdx.y * 64; i0 < live_rows * (HDP / 4); i0 += 64 * gridDim.y) {
    const int i = min(i0 + lane, live_rows * (HDP / 4) - 1);
    const int r = i / (HDP / 4), d = 4 * (i % (HDP / 4));
    float top = -__builtin_inff(), l = 0.0f;
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    // A factor for a maximum against a higher one; a piece without keys has none (0, not exp2(-inf - -inf)).
    auto factor = [](float m, float high) { return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - high); };
    // A NaN among a piece's scores is in its sum, whatever its maximum says.
    auto sum = [](float l, float f) { return l != l ? l : f * l; };
    for (int w0 = first + wave; w0 <= pc.last; w0 += kJoinWaves * kJoinAhead) {
      float m[kJoinAhead], lw[kJoinAhead];
      float4_t x[kJoinAhead];
      float high = top;
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int w = min(w0 + kJoinWaves * j, pc.last);
        const float* const p = ws + (size_t)(2 * w + (w == first ? 1 : 0)) * STRIDE;
        m[j] = p[ROWS * HDP + r];
        lw[j] = p[ROWS * HDP + ROWS + r];
        x[j] = *reinterpret_cast<const float4_t*>(p + r * HDP + d);
      }
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j)
        if (w0 + kJoinWaves * j <= pc.last) high = fmaxf(high, m[j]);
      const float old = factor(top, high);
      l = sum(l, old);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scaled(v[e], old);
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        if (w0 + kJoinWaves * j > pc.last) break;
        const float f = factor(m[j], high);
        l += sum(lw[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += scaled(x[j][e], f);
      }
      top = high;
    }
    __syncthreads();  // the last values have been read
    stat[0][wave][lane] = top;
    stat[1][wave][lane] = l;
    parts[wave][lane] = v;
    __syncthreads();
    if (wave != 0) continue;
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) top = fmaxf(top, stat[0][w][lane]);
    l = 0.0f;
    v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      const float f = factor(stat[0][w][lane], top);
      l += sum(stat[1][w][lane], f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += scaled(parts[w][lane][e], f);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int row = pc.row0 + r, tok = row / rep, head = pc.kv * rep + (row - tok * rep);
    if (d < a.head_dim && i0 + lane < live_rows * (HDP / 4))
      store_global((E*)a.out + (size_t)(tok0 + tok) * a.out_token + (size_t)head * a.out_head + d,
                   u32x2{Elem<E>::pack(v[0] * inv, v[1] * inv), Elem<E>::pack(v[2] * inv, v[3] * inv)});
  }
}
}  // namespace

}  // namespace kf
