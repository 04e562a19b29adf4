// pd_fp4_attend.cu -- launcher of the attention over 4-bit pages (pd_fp4_attend.cuh).
#include "pd_fp4_attend.cuh"

#include "paged_decode.h"

namespace pd {

namespace {

// Warps per CTA, one CTA per SM: 16 where a thread's columns fit 128 registers, 8 at head_dim 256
// (its accumulators and query fragments alone are 96). Measured at 32 rows of 8192 tokens, head_dim
// 128, with an earlier inner loop: 71 us with 16 warps, 76 with 12, 86 with 8; at head_dim 256, 61 skewed
// rows: 28.4 us with 8, 31.1 with 10 (which spill), and 12 leave no room for the rings.
template <int D>
struct Warps {
  static constexpr int NW = D == 256 ? 8 : 16;
};

constexpr int kMaxSmem = 232448 - 1024;  // per CTA, less the kernel's static part

template <typename T, int D>
cudaError_t launch_t(const Fp4AttendParams& p, int sms, cudaStream_t stream) {
  constexpr int NW = Warps<D>::NW;
  auto fn = fp4::pd_fp4_attend_kernel<T, D, NW>;
  static_assert(fp4::smem_layout(fp4::MAX_ROWS, NW, fp4::COLS, D, 2).bytes <= kMaxSmem, "the longest launch fits");
  const int64_t most = int64_t(p.max_seqlen_q) * p.group;
  const int cols = int(most < fp4::COLS ? most : fp4::COLS);
  int stages = 4;  // as many as shared memory holds
  while (stages > 2 && fp4::smem_layout(p.batch, NW, cols, D, stages).bytes > kMaxSmem) --stages;
  const int bytes = fp4::smem_layout(p.batch, NW, cols, D, stages).bytes;
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, kMaxSmem, raised);
  if (err != cudaSuccess) return err;
  fn<<<dim3(unsigned(sms)), NW * 32, bytes, stream>>>(p, stages, cols);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_d(const Fp4AttendParams& p, int head_dim, int sms, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_t<T, 64>(p, sms, stream);
    case 128: return launch_t<T, 128>(p, sms, stream);
    case 256: return launch_t<T, 256>(p, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int fp4_max_rows() { return fp4::MAX_ROWS; }

// [counters: one per CTA, 256-byte multiple | two partials per CTA]
size_t fp4_counter_bytes(int sms) { return (size_t(sms) * 4 + 255) / 256 * 256; }
size_t fp4_workspace_bytes(int head_dim, int sms) {
  return fp4_counter_bytes(sms) + size_t(sms) * 2 * fp4::partial_floats(head_dim) * 4;
}

cudaError_t launch_fp4_attend(const Fp4AttendParams& p, int dtype, int head_dim, int sms, cudaStream_t stream) {
  return dtype == PD_BF16 ? launch_d<__nv_bfloat16>(p, head_dim, sms, stream)
                          : launch_d<__half>(p, head_dim, sms, stream);
}

}  // namespace pd
