// attention.cu -- attention of new tokens over a paged key/value cache: which
// kernel a call takes, and its launch.
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
  p.least_units = 4;
  // Two blocks an SM, or what the longest possible work fills.
  return launch_after(attn_rows_kernel<T, FP8, D>, dim3(2 * num_sms), dim3(128), K::kSmem, 1, stream, p);
}

template <typename T, bool FP8, int D>
cudaError_t launch_tiles(AttnParams p, int num_sms, cudaStream_t stream) {
  using K = TilesKernel<T, FP8, D>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(attn_tiles_kernel<T, FP8, D>), K::kSmem, &allowed);
  if (e != cudaSuccess) return e;
  p.least_units = 2;
  return launch_after(attn_tiles_kernel<T, FP8, D>, dim3(num_sms), dim3(K::kThreads), K::kSmem, 1, stream, p);
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

size_t attn_counter_bytes(int num_sms) { return ((size_t)num_sms * 2 * 4 + 255) / 256 * 256; }
size_t attn_part_bytes(int num_sms, int head_dim) {
  const size_t rows = 2 * (size_t)(head_dim * 16 + 32), tiles = 2 * (size_t)(head_dim * 128 + 256);
  static_assert(RowsKernel<__half, false, 64>::kPartFloats == 64 * 16 + 32 &&
                    TilesKernel<__half, false, 64>::kPartFloats == 64 * 128 + 256,
                "a block's parts");
  return (size_t)num_sms * 2 * (rows > tiles ? rows : tiles) * 4;
}

cudaError_t launch_attention(const AttnParams& p, int num_sms, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  if (p.bf16)
    return fp8 ? launch_typed<__nv_bfloat16, true>(p, num_sms, stream)
               : launch_typed<__nv_bfloat16, false>(p, num_sms, stream);
  return fp8 ? launch_typed<__half, true>(p, num_sms, stream) : launch_typed<__half, false>(p, num_sms, stream);
}

}  // namespace b2g
