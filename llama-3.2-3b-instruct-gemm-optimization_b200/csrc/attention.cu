// attention.cu -- attention of new tokens over a paged key/value cache: which
// kernel a call takes, and its launch.
#include <algorithm>
#include <type_traits>

#include "attn_rows.cuh"
#include "attn_tiles.cuh"

namespace b2g {
namespace {

template <typename T, bool FP8, int D>
cudaError_t launch_rows(AttnParams p, int num_sms, cudaStream_t stream) {
  using K = RowsKernel<T, FP8, D>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(attn_rows_kernel<T, FP8, D>), K::kSmem, &allowed);
  if (e != cudaSuccess) return e;
  // Two units a block at least: one sequence of 1000 tokens 11.2 us (13.2 with
  // four), of 4001 15.8 (16.5).
  p.least_units = 2;
  return launch_after(attn_rows_kernel<T, FP8, D>, dim3(K::kBlocks * num_sms), dim3(128), K::kSmem, 1, stream, p);
}

// A 16-bit cache as (dim, row, head, page); loads of 64 elements by `rows`.
bool encode_cache(CUtensorMap* map, void* base, const b2g_kv_cache& c, int rows) {
  const EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads,
                              (cuuint64_t)c.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c.stride_token * 2, (cuuint64_t)c.stride_head * 2,
                                 (cuuint64_t)c.stride_page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool FP8, int D>
cudaError_t launch_tiles(AttnParams p, int num_sms, cudaStream_t stream) {
  using K = TilesKernel<T, FP8, D>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(attn_tiles_kernel<T, FP8, D>), K::kSmem, &allowed);
  if (e != cudaSuccess) return e;
  // Four units a block at least (3 chunks of up to 1672 tokens, 4 heads: 59 us,
  // 65 with two), one if the items are short (2 chunks of 640 with a window of
  // 100: 35 us, 53 with two).
  p.least_units = 4;
  AttnTilesParams a;
  a.p = p;
  a.tma.box_rows = 0;
  // Pages that divide a unit, or that units divide, in 8-row steps (the
  // swizzle's period): whole units by TMA.  Other pages, 8-bit caches (they
  // are widened on the way) and strides beyond a tensor map's go by 16-byte
  // copies.
  const int page = p.c.page_size;
  if (!FP8 && page % 8 == 0 && (K::kUnit % page == 0 || page % K::kUnit == 0)) {
    const int rows = page < K::kUnit ? page : K::kUnit;
    if (encode_cache(&a.tma.k, p.c.k, p.c, rows) && encode_cache(&a.tma.v, p.c.v, p.c, rows)) a.tma.box_rows = rows;
  }
  return launch_after(attn_tiles_kernel<T, FP8, D>, dim3(num_sms), dim3(K::kThreads), K::kSmem, 1, stream, a);
}

template <typename T, bool FP8, int D>
cudaError_t launch_sized(const AttnParams& p, int num_sms, cudaStream_t stream) {
  // One 16-row tile holds every sequence's rows of a k/v head: the kernel
  // that reads the cache once and no more; else the tensor-memory kernel.
  if ((long long)p.b.max_q * p.group <= 16) return launch_rows<T, FP8, D>(p, num_sms, stream);
  return launch_tiles<T, FP8, D>(p, num_sms, stream);
}

template <typename T, bool FP8>
cudaError_t launch_typed(const AttnParams& p, int num_sms, cudaStream_t stream) {
  if (p.c.head_dim == 128) return launch_sized<T, FP8, 128>(p, num_sms, stream);
  return launch_sized<T, FP8, 64>(p, num_sms, stream);
}

}  // namespace

// A counter a block of the rows kernel, and a tile and block (one an SM) of the
// tiles kernel; two parts for each.
size_t attn_counter_bytes(int num_sms) {
  static_assert(RowsKernel<__half, false, 64>::kBlocks <= kAttnBlocks && RowsKernel<__half, true, 128>::kBlocks <= kAttnBlocks,
                "a block's counters and parts");
  return ((size_t)num_sms * std::max(kAttnBlocks, kAttnTiles) * 4 + 255) / 256 * 256;
}
size_t attn_part_bytes(int num_sms, int head_dim) {
  const size_t rows = kAttnBlocks * (size_t)(head_dim * 16 + 32), tiles = kAttnTiles * (size_t)(head_dim * 128 + 256);
  static_assert(RowsKernel<__half, false, 64>::kPartFloats == 64 * 16 + 32 &&
                    TilesKernel<__half, false, 64>::kPartFloats == 64 * 128 + 256 &&
                    TilesKernel<__half, false, 64>::kRows == kAttnTiles * TilesKernel<__half, false, 64>::kTile,
                "a block's parts");
  return (size_t)num_sms * 2 * std::max(rows, tiles) * 4;
}

cudaError_t launch_attention(const AttnParams& p, int num_sms, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  if (p.bf16)
    return fp8 ? launch_typed<__nv_bfloat16, true>(p, num_sms, stream)
               : launch_typed<__nv_bfloat16, false>(p, num_sms, stream);
  return fp8 ? launch_typed<__half, true>(p, num_sms, stream) : launch_typed<__half, false>(p, num_sms, stream);
}

}  // namespace b2g
