// Router balance loss, z-loss and per-expert counts, with the gradient.
//
//   c_e = #slots of counted tokens that name expert e,  f_e = c_e / max(1, sum c),
//   p_t = softmax(logits_t),  S_t = sum_e f_e p_te,  n = max(1, #counted tokens)
//   loss = E/n * sum_t S_t + z/n * sum_t lse_t^2
//   dloss/dlogits_te = p_te * (E/n * (f_e - S_t) + 2 z/n * lse_t)
//
// f depends on the slots alone, so a first small kernel counts them and the second reads
// every logit once and writes its gradient at once: the logits are not read again in a
// backward pass.  The counts are integers and the loss is summed in a fixed order, so
// results do not depend on the order in which CTAs run.
#include "common.cuh"

namespace fk {
namespace {

constexpr int kMaxExperts = 256;
constexpr int kCountCtas = 64;       // partial histograms that every CTA of the second kernel adds up
constexpr int kCountThreads = 256;
constexpr int kCountStride = kMaxExperts + 2;  // E counts, then the counted tokens, then bad slots
constexpr int kMainThreads = 256;
constexpr int kMainCtasPerSm = 8;

struct Workspace {
  int* part;      // [kCountCtas][kCountStride]
  double2* sums;  // [main grid] (sum S, sum lse^2)
  unsigned* ticket;
};

inline size_t ws_bytes() {
  return (size_t)kCountCtas * kCountStride * sizeof(int) +
         (size_t)num_sms() * kMainCtasPerSm * sizeof(double2) + 16;
}
inline Workspace ws_split(void* p) {
  Workspace w;
  w.sums = static_cast<double2*>(p);
  char* q = static_cast<char*>(p) + (size_t)num_sms() * kMainCtasPerSm * sizeof(double2);
  w.ticket = reinterpret_cast<unsigned*>(q);
  w.part = reinterpret_cast<int*>(q + 16);
  return w;
}

// Slots are counted in shared memory and leave as one partial histogram per CTA.
__global__ void __launch_bounds__(kCountThreads) balance_count(
    const int64_t* __restrict__ idx, const uint8_t* __restrict__ mask, int64_t n_rows, int k,
    int n_experts, int* __restrict__ part, unsigned* __restrict__ ticket) {
  __shared__ int hist[kCountStride];
  for (int i = threadIdx.x; i < n_experts + 2; i += blockDim.x) hist[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  __syncthreads();
  int tokens = 0, bad = 0;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < n_rows; t += step) {
    if (mask && !mask[t]) continue;
    ++tokens;
    for (int j = 0; j < k; ++j) {
      const int64_t e = idx[t * k + j];
      if (e >= n_experts) ++bad;
      else if (e >= 0) atomicAdd(&hist[e], 1);
    }
  }
  if (tokens) atomicAdd(&hist[n_experts], tokens);
  if (bad) atomicAdd(&hist[n_experts + 1], bad);
  __syncthreads();
  for (int i = threadIdx.x; i < n_experts + 2; i += blockDim.x)
    part[(int64_t)blockIdx.x * kCountStride + i] = hist[i];
}

// One warp per token, lane l holds experts l, l+32, ...
template <typename T>
__global__ void __launch_bounds__(kMainThreads) balance_main(
    const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ mask,
    int64_t n_rows, int n_experts, float z_coef, float loss_scale, const int* __restrict__ part,
    int count_ctas, T* __restrict__ grad, int64_t* __restrict__ counts, double2* __restrict__ sums,
    unsigned* __restrict__ ticket, float* __restrict__ loss) {
  constexpr int kPer = kMaxExperts / 32;
  __shared__ int tot[kCountStride];
  __shared__ float f[kMaxExperts];
  __shared__ double2 red[kMainThreads / 32];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = kMainThreads / 32;
  for (int i = threadIdx.x; i < n_experts + 2; i += blockDim.x) {
    int c = 0;
    for (int g = 0; g < count_ctas; ++g) c += part[(int64_t)g * kCountStride + i];
    tot[i] = c;
  }
  __syncthreads();
  int64_t slots = 0;
  for (int e = 0; e < n_experts; ++e) slots += tot[e];
  const bool bad = tot[n_experts + 1] != 0;
  const float inv_slots = 1.0f / (float)(slots < 1 ? 1 : slots);
  const float n = (float)(tot[n_experts] < 1 ? 1 : tot[n_experts]);
  for (int e = threadIdx.x; e < n_experts; e += blockDim.x) {
    f[e] = bad ? __int_as_float(0x7fc00000) : (float)tot[e] * inv_slots;
    if (blockIdx.x == 0) counts[e] = tot[e];
  }
  __syncthreads();
  const float ce = (float)n_experts * loss_scale / n, cz = 2.f * z_coef * loss_scale / n;
  double sum_s = 0.0, sum_z = 0.0;
  for (int64_t t = (int64_t)blockIdx.x * nwarps + warp; t < n_rows;
       t += (int64_t)gridDim.x * nwarps) {
    T* out = grad ? grad + t * n_experts : nullptr;
    if (mask && !mask[t]) {
      if (out)
        for (int e = lane; e < n_experts; e += 32) out[e] = Elt<T>::from_f(0.f);
      continue;
    }
    const T* row = logits + t * stride;
    float v[kPer];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < n_experts ? Elt<T>::to_f(row[e]) : -INFINITY;
      m = fmaxf(m, v[i]);  // a NaN is passed over here and comes back in the sum
    }
    m = warp_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float z = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      v[i] = expf(v[i] - base);
      z += v[i];
      s = fmaf(v[i], e < n_experts ? f[e] : 0.f, s);
    }
    z = warp_sum(z);
    s = warp_sum(s);
    // A row of -inf alone has no probabilities: it adds nothing and gets no gradient.
    const float inv = z == 0.f ? 0.f : 1.0f / z;
    const float lse = z == 0.f ? 0.f : base + logf(z);
    s *= inv;
    sum_s += (double)s;
    sum_z += (double)lse * (double)lse;
    if (out) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        if (e < n_experts) out[e] = Elt<T>::from_f(v[i] * inv * fmaf(ce, f[e] - s, cz * lse));
      }
    }
  }
  if (lane == 0) red[warp] = make_double2(sum_s, sum_z);
  __syncthreads();
  if (threadIdx.x == 0) {
    double2 a = make_double2(0.0, 0.0);
    for (int i = 0; i < nwarps; ++i) {
      a.x += red[i].x;
      a.y += red[i].y;
    }
    sums[blockIdx.x] = a;
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (last && threadIdx.x == 0) {
    __threadfence();
    double a = 0.0, b = 0.0;
    for (unsigned i = 0; i < gridDim.x; ++i) {
      a += __ldcg(&sums[i].x);
      b += __ldcg(&sums[i].y);
    }
    *loss = (float)(((double)n_experts * a + (double)z_coef * b) / (double)n);
  }
}

template <typename T>
int fwd_t(const void* logits, int64_t stride, const int64_t* idx, const uint8_t* mask,
          int64_t n_rows, int n_experts, int k, float z_coef, float loss_scale, void* grad,
          int64_t* counts, float* loss, void* workspace, cudaStream_t st) {
  const Workspace ws = ws_split(workspace);
  int64_t g = (n_rows + kCountThreads - 1) / kCountThreads;
  const int count_ctas = (int)(g < 1 ? 1 : g > kCountCtas ? kCountCtas : g);
  balance_count<<<count_ctas, kCountThreads, 0, st>>>(idx, mask, n_rows, k, n_experts, ws.part,
                                                      ws.ticket);
  int s = launch_status("fk_moe_balance(count)");
  if (s != FK_OK) return s;
  const int64_t want = (n_rows + kMainThreads / 32 - 1) / (kMainThreads / 32);
  const int64_t most = (int64_t)num_sms() * kMainCtasPerSm;
  const int grid = (int)(want < 1 ? 1 : want > most ? most : want);
  balance_main<T><<<grid, kMainThreads, 0, st>>>(
      static_cast<const T*>(logits), stride, mask, n_rows, n_experts, z_coef, loss_scale, ws.part,
      count_ctas, static_cast<T*>(grad), counts, ws.sums, ws.ticket, loss);
  return launch_status("fk_moe_balance");
}

}  // namespace
}  // namespace fk

extern "C" int fk_moe_balance_workspace_size(size_t* bytes) {
  FK_CHECK_ARG(bytes != nullptr, "fk_moe_balance_workspace_size: null output");
  *bytes = fk::ws_bytes();
  return FK_OK;
}

extern "C" int fk_moe_balance(const void* logits, int64_t row_stride, const int64_t* idx,
                              const uint8_t* token_mask, int64_t n_rows, int n_experts, int k,
                              float z_coef, float loss_scale, void* grad, int64_t* counts,
                              float* loss, void* workspace, size_t workspace_bytes, int dtype,
                              void* stream) {
  FK_CHECK_ARG(n_rows >= 0 && n_experts >= 1 && k >= 0, "fk_moe_balance: bad shape");
  if (n_experts > fk::kMaxExperts)
    return fk::fail(FK_ERR_UNSUPPORTED, "fk_moe_balance: n_experts=%d exceeds %d", n_experts,
                    fk::kMaxExperts);
  FK_CHECK_ARG(n_rows * (int64_t)(k < 1 ? 1 : k) < (int64_t)1 << 31,
               "fk_moe_balance: more than 2^31 slots");
  FK_CHECK_ARG(row_stride >= n_experts, "fk_moe_balance: stride < n_experts");
  FK_CHECK_ARG(fk::valid_dtype(dtype), "fk_moe_balance: bad dtype code %d", dtype);
  FK_CHECK_ARG(counts && loss, "fk_moe_balance: null pointer");
  FK_CHECK_ARG(n_rows == 0 || (logits && (idx || k == 0)), "fk_moe_balance: null pointer");
  if (workspace == nullptr || workspace_bytes < fk::ws_bytes() || !fk::aligned16(workspace))
    return fk::fail(FK_ERR_WORKSPACE, "fk_moe_balance: need %zu aligned workspace bytes, got %zu",
                    fk::ws_bytes(), workspace_bytes);
  FK_DISPATCH_DTYPE(dtype, return fk::fwd_t<scalar_t>(logits, row_stride, idx, token_mask, n_rows,
                                                      n_experts, k, z_coef, loss_scale, grad,
                                                      counts, loss, workspace,
                                                      fk::as_stream(stream)));
  return FK_OK;
}
