// attention.cu -- attention of new tokens over a paged key/value cache: which
// kernel a call takes, and its launch.
#include <type_traits>

#include "attn_rows.cuh"

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

template <typename T, bool FP8>
cudaError_t launch_typed(const AttnParams& p, int num_sms, cudaStream_t stream) {
  if (p.c.head_dim == 128) return launch_rows<T, FP8, 128>(p, num_sms, stream);
  return launch_rows<T, FP8, 64>(p, num_sms, stream);
}

}  // namespace

size_t attn_counter_bytes(int num_sms) { return ((size_t)num_sms * 2 * 4 + 255) / 256 * 256; }
size_t attn_part_bytes(int num_sms, int head_dim) {
  return (size_t)num_sms * 2 * 2 * RowsKernel<__half, false, 128>::kPartFloats * 4;
}

cudaError_t launch_attention(const AttnParams& p, int num_sms, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  if (p.bf16)
    return fp8 ? launch_typed<__nv_bfloat16, true>(p, num_sms, stream)
               : launch_typed<__nv_bfloat16, false>(p, num_sms, stream);
  return fp8 ? launch_typed<__half, true>(p, num_sms, stream) : launch_typed<__half, false>(p, num_sms, stream);
}

}  // namespace b2g
