// Gradients that a forward pass wrote for one grad_output, brought to another one.
#include "common.cuh"

namespace fk {
namespace {

// Every CTA reads grad_output and leaves where it is the expected one: the launch then costs
// its 2 us and touches nothing.
template <typename T>
__global__ void __launch_bounds__(512) grad_rescale(T* grad, int64_t stride, int64_t rows,
                                                    int64_t cols,
                                                    const float* __restrict__ grad_output,
                                                    float expected, int flat) {
  const float go = *grad_output;
  if (go == expected) return;
  const float s = go / expected;
  constexpr int VN = 16 / (int)sizeof(T);
  if (flat) {  // contiguous and aligned: 16-byte packets
    const int64_t n = rows * cols, packets = n / VN;
    const int64_t me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t v = me; v < packets; v += step) {
      Vec16<T> p = ld_stream(grad + v * VN);
#pragma unroll
      for (int e = 0; e < VN; ++e) p.e[e] = Elt<T>::from_f(Elt<T>::to_f(p.e[e]) * s);
      st_stream(grad + v * VN, p);
    }
    for (int64_t i = packets * VN + me; i < n; i += step)
      grad[i] = Elt<T>::from_f(Elt<T>::to_f(grad[i]) * s);
    return;
  }
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x)
      grad[r * stride + c] = Elt<T>::from_f(Elt<T>::to_f(grad[r * stride + c]) * s);
}

}  // namespace
}  // namespace fk

extern "C" int fk_grad_rescale(void* grad, int64_t row_stride, int64_t rows, int64_t cols,
                               const float* grad_output, float expected, int dtype,
                               void* stream) {
  FK_CHECK_ARG(rows >= 0 && cols >= 0, "fk_grad_rescale: negative shape");
  FK_CHECK_ARG(fk::valid_dtype(dtype), "fk_grad_rescale: bad dtype code %d", dtype);
  FK_CHECK_ARG(expected == expected && expected != 0.f, "fk_grad_rescale: expected is 0 or NaN");
  if (rows == 0 || cols == 0) return FK_OK;
  FK_CHECK_ARG(row_stride >= cols, "fk_grad_rescale: stride < cols");
  FK_CHECK_ARG(grad && grad_output, "fk_grad_rescale: null pointer");
  const int flat = fk::aligned16(grad) && (row_stride == cols || rows == 1);
  const int64_t want = flat ? (rows * cols / 512 + 1) / 4 + 1 : rows;
  const int64_t most = (int64_t)fk::num_sms() * 4;
  const unsigned grid = (unsigned)(want < most ? want : most);
  FK_DISPATCH_DTYPE(dtype, {
    fk::grad_rescale<scalar_t><<<grid, 512, 0, fk::as_stream(stream)>>>(
        static_cast<scalar_t*>(grad), row_stride, rows, cols, grad_output, expected, flat);
  });
  return fk::launch_status("fk_grad_rescale");
}
