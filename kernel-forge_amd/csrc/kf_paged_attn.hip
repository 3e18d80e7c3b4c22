// Launches of the attention of few rows per request (kf_few_rows.h), and where its work is cut.
#include <algorithm>

#include "kf_few_rows.h"
#include "kf_launch.h"

namespace kf {
namespace {

template <class E, class C, bool CUT>
__global__ __launch_bounds__(C::THREADS) void few_rows_kernel(AttnArgs a, int rep, int max_rows, float scale_log2, float* ws,
                                                              Piece* pieces) {
  __shared__ FewShared<C> sh;
  few_rows_stretch<E, C, CUT>(a, sh, (int)blockIdx.x, (int)gridDim.x, rep, max_rows, scale_log2, ws, pieces);
}

template <class E, int HDP, int MT, int WAVES>
hipError_t launch(const AttnArgs& a, const FewPlan& p, int max_rows, void* ws, hipStream_t stream) {
  using C = FewConfig<HDP, MT, WAVES>;
  const int rep = a.heads / a.kv_heads;
  const float scale_log2 = a.scale * 1.44269504088896340736f;
  if (!p.cut) {
    few_rows_kernel<E, C, false><<<p.grid, C::THREADS, 0, stream>>>(a, rep, max_rows, scale_log2, nullptr, nullptr);
    return hipGetLastError();
  }
  float* const parts = static_cast<float*>(ws);
  Piece* const pieces = reinterpret_cast<Piece*>(parts + (size_t)2 * p.grid * C::ROWS * (HDP + 2));
  few_rows_kernel<E, C, true><<<p.grid, C::THREADS, 0, stream>>>(a, rep, max_rows, scale_log2, parts, pieces);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  join_pieces_kernel<E, HDP, C::ROWS><<<join_grid<HDP, C::ROWS>(p.grid), 64 * kJoinWaves, 0, stream>>>(a, rep, parts, pieces);
  return hipGetLastError();
}

template <class E, int HDP>
hipError_t launch_rows(const AttnArgs& a, const FewPlan& p, int max_rows, void* ws, hipStream_t stream) {
  if constexpr (HDP == 256) {  // one row tile of 256 dims fills the registers, two wavefronts the buffers
    return launch<E, HDP, 1, 2>(a, p, max_rows, ws, stream);
  } else {
    if (p.waves == 2)
      return p.row_tiles == 2 ? launch<E, HDP, 2, 2>(a, p, max_rows, ws, stream)
                              : launch<E, HDP, 1, 2>(a, p, max_rows, ws, stream);
    return p.row_tiles == 2 ? launch<E, HDP, 2, 4>(a, p, max_rows, ws, stream)
                            : launch<E, HDP, 1, 4>(a, p, max_rows, ws, stream);
  }
}

template <class E>
hipError_t launch_dim(const AttnArgs& a, const FewPlan& p, int max_rows, void* ws, hipStream_t stream) {
  if (a.head_dim <= 64) return launch_rows<E, 64>(a, p, max_rows, ws, stream);
  if (a.head_dim <= 128) return launch_rows<E, 128>(a, p, max_rows, ws, stream);
  return launch_rows<E, 256>(a, p, max_rows, ws, stream);
}

}  // namespace

FewPlan few_rows_plan(const AttnArgs& a, int64_t rows, int max_rows, int cu_count, bool beside) {
  FewPlan p;
  p.row_tiles = beside || (a.head_dim <= 128 && rows > 16) ? 2 : 1;
  // By the rows of all requests, and by the most that a request of this kernel's has.
  const int64_t tile = 16 * p.row_tiles;
  const int64_t items = std::min((int64_t)a.tokens * (a.heads / a.kv_heads) / tile + a.seqs,
                                 a.seqs * ((max_rows + tile - 1) / tile)) * a.kv_heads;
  // The lengths are on the device, so plans go by what the table has room for.  Tables of 131072 tokens in place of tight
  // ones, us: 16 requests of up to 450 tokens 8.5 -> 11.2, 128 of 50 .. 900 (8 KV heads of 128) 33 -> 41.
  const int64_t keys = (int64_t)a.table_width << a.log2_block;
  // A CU holds one workgroup of four wavefronts or two of two, one of which then copies while the other begins or ends an
  // item.  That pays where there are an item or more for each CU and they are short; otherwise the second
  // workgroup's pieces only cost.  Four / two, us: 128 requests of up to 700 tokens, 8 KV heads of 128, 44 / 35, of
  // up to 2000 82 / 85, 4 heads of 64 34 / 30, of up to 6000 66 / 66; 16 of up to 700, 4 of 64, 11.5 / 12.5.
  p.waves = beside || a.head_dim > 128 || (items >= cu_count && keys * (a.head_dim <= 64 ? 64 : 128) <= 1 << 17) ? 2 : 4;
  const int unit = 32 * p.waves, fits = (a.head_dim <= 128 && p.waves == 2 && !beside ? 2 : 1) * cu_count;
  const int64_t key_units = (keys + unit - 1) / unit;
  // Up to 512 keys are worked off whole, without the second launch.  Whole / cut, us: 16 requests of up to 450 tokens
  // 8.7 / 11.2, of up to 900 11.3 / 11.8, of up to 1900 17.2 / 12.8; one of 900 15.6 / 11.5.
  p.cut = key_units * unit > 512;
  p.most_units = items * (key_units + kFewItem);
  p.grid = (int)std::min<int64_t>(fits, p.cut ? p.most_units : items);
  return p;
}

size_t few_rows_workspace_bytes(int head_dim, const FewPlan& p) {
  if (!p.cut) return 0;
  const int padded = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  return (size_t)p.grid * (2 * sizeof(float) * 16 * p.row_tiles * (padded + 2) + sizeof(Piece));
}

hipError_t few_rows_launch(const AttnArgs& a, bool bf16, const FewPlan& p, int max_rows, void* ws, hipStream_t stream) {
  return bf16 ? launch_dim<bhalf_t>(a, p, max_rows, ws, stream) : launch_dim<half_t>(a, p, max_rows, ws, stream);
}

}  // namespace kf
