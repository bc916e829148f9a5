// Distillation from a teacher's top logits, optionally mixed with the hard label: loss and
// gradient.  Per row, over the used slots j (id i_j >= 0, teacher logit t_j):
//
//   p = softmax(t / T) over the slots,  q = softmax(s / T) over the vocabulary
//   soft = T^2 * sum_j p_j (log p_j - s_{i_j}/T + lse(s/T)),  hard = lse(s) - s_y
//   loss = 1/n * sum_rows [(1-a) soft + a hard]
//   dloss/ds_c = 1/n * [(1-a) T (q_c - P_c) + a (softmax(s)_c - [c = y])],
//   P_c = sum of the p_j whose id is c.
//
// The teacher's side of a row is small and is done first, by one warp per row: it leaves a
// list of (id, P) with every id once and the label's entry last, the row's sum p log p, and
// partial counts of the rows that count (n).  The second kernel then needs every logit once
// for the two sums and once for its gradient, and the gradient at the listed ids is computed
// from the logit itself, in 32 bits, and rounded once.
#include "common.cuh"

namespace fk {
namespace {

constexpr int kMaxSlots = 1024;
constexpr int kTeacherWarps = 8;
constexpr int kTeacherCtas = 64;   // partial counts that every CTA of the second kernel adds up
constexpr int kRowThreads = 256;
constexpr int kRowCtasPerSm = 4;
// Row states.
constexpr int kSkip = 0, kSoft = 1, kHard = 2, kBad = 4;

struct Workspace {
  int2* valid;       // [kTeacherCtas] (rows that count, rows with an id out of range)
  unsigned* ticket;
  float* loss_rows;  // [n_rows]
  float* entropy;    // [n_rows]  sum p log p
  int* state;        // [n_rows]
  int* ids;          // [n_rows][list]  -1 = empty
  float* probs;      // [n_rows][list]
};
inline size_t align16(size_t n) { return (n + 15) / 16 * 16; }
inline size_t ws_layout(void* base, int64_t n_rows, int k, Workspace* w) {
  char* p = static_cast<char*>(base);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* q = p + at;
    at += align16(bytes);
    return q;
  };
  const size_t n = (size_t)n_rows, list = (size_t)k + 1;
  w->valid = reinterpret_cast<int2*>(take(kTeacherCtas * 8));
  w->ticket = reinterpret_cast<unsigned*>(take(4));
  w->loss_rows = reinterpret_cast<float*>(take(n * 4));
  w->entropy = reinterpret_cast<float*>(take(n * 4));
  w->state = reinterpret_cast<int*>(take(n * 4));
  w->ids = reinterpret_cast<int*>(take(n * list * 4));
  w->probs = reinterpret_cast<float*>(take(n * list * 4));
  return at;
}

// ------------------------------------------------------------------ teacher -------------
// Shared memory per warp: ids[k], p[k], and a hash table that finds ids standing twice.
template <typename T>
__global__ void __launch_bounds__(kTeacherWarps * 32) distill_teacher(
    const int64_t* __restrict__ idx, const T* __restrict__ top, int k, int table,
    const int64_t* __restrict__ targets, int64_t ignore_index, int64_t n_rows, int64_t n_cols,
    float inv_t, Workspace ws) {
  extern __shared__ int smem[];
  __shared__ int valid_rows, bad_rows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* ids = smem + warp * (2 * k + table);
  float* p = reinterpret_cast<float*>(ids + k);
  int* hash = ids + 2 * k;
  if (threadIdx.x == 0) {
    valid_rows = bad_rows = 0;
    if (blockIdx.x == 0) *ws.ticket = 0;
  }
  __syncthreads();
  const int list = k + 1;
  for (int64_t row = (int64_t)blockIdx.x * kTeacherWarps + warp; row < n_rows;
       row += (int64_t)gridDim.x * kTeacherWarps) {
    const int64_t y = targets ? targets[row] : -1;
    const bool ignored = targets && y == ignore_index;
    bool bad = targets && !ignored && (y < 0 || y >= n_cols);
    for (int i = lane; i < table; i += 32) hash[i] = -1;
    __syncwarp();
    float m = -INFINITY;
    bool twice = false, nan = false;
    for (int j = lane; j < k; j += 32) {
      const int64_t id = idx[row * k + j];
      const bool out = id >= n_cols;
      bad = bad || (out && !ignored);
      const int c = (id < 0 || out) ? -1 : (int)id;
      const float v = Elt<T>::to_f(top[row * k + j]);
      ids[j] = c;
      p[j] = v;
      if (c >= 0) {
        m = fmaxf(m, v);
        nan = nan || v != v;
        unsigned at = ((unsigned)c * 2654435761u) & (unsigned)(table - 1);
        for (;;) {  // at most k ids in a table of at least 2k places: a free one is found
          const int old = atomicCAS(&hash[at], -1, c);
          if (old == -1) break;
          if (old == c) {
            twice = true;
            break;
          }
          at = (at + 1) & (unsigned)(table - 1);
        }
      }
    }
    bad = __any_sync(0xffffffffu, bad);
    twice = __any_sync(0xffffffffu, twice);
    m = warp_max(m);
    float z = 0.f;
    for (int j = lane; j < k; j += 32)
      if (ids[j] >= 0) z += expf((p[j] - m) * inv_t);  // m = -inf: NaN, and the row has no teacher
    z = warp_sum(z);
    const bool held = m != -INFINITY || __any_sync(0xffffffffu, nan);
    const float lz = logf(z), inv_z = 1.0f / z;
    float ent = 0.f;
    for (int j = lane; j < k; j += 32) {
      float pj = 0.f;
      if (held && ids[j] >= 0) {
        const float d = (p[j] - m) * inv_t;
        pj = expf(d) * inv_z;
        if (pj > 0.f) ent = fmaf(pj, d - lz, ent);
        else if (pj != pj) ent = pj;
      }
      p[j] = pj;
    }
    ent = warp_sum(ent);
    __syncwarp();
    int state = kSkip;
    if (!ignored && bad) state = kBad;
    else if (!ignored) state = (held ? kSoft : 0) | (targets ? kHard : 0);
    // The list: every id once, at its first slot, with the sum of its probabilities; the
    // label's at the end.
    float py = 0.f;
    for (int j = lane; j < k; j += 32) {
      int c = ids[j];
      float pj = p[j];
      if (twice && c >= 0) {
        pj = 0.f;
        int first = j;
        for (int i = 0; i < k; ++i)
          if (ids[i] == c) {
            if (i < first) first = i;
            pj += p[i];
          }
        if (first != j) c = -1;
      }
      if ((state & kHard) && c == (int)y && c >= 0) {
        py += pj;
        c = -1;
      }
      if (!held) c = -1;
      ws.ids[row * list + j] = c;
      ws.probs[row * list + j] = c >= 0 ? pj : 0.f;
    }
    py = warp_sum(py);
    if (lane == 0) {
      ws.ids[row * list + k] = (state & kHard) ? (int)y : -1;
      ws.probs[row * list + k] = py;
      ws.entropy[row] = ent;
      ws.state[row] = state;
      if (state != kSkip) atomicAdd(&valid_rows, 1);
      if (state == kBad) atomicAdd(&bad_rows, 1);
    }
    __syncwarp();
  }
  __syncthreads();
  if (threadIdx.x == 0) ws.valid[blockIdx.x] = make_int2(valid_rows, bad_rows);
}

// ------------------------------------------------------------------ rows ----------------
__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float m = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) m = fmaxf(m, red[i]);
  return m;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
  return s;
}

struct RowArgs {
  const int2* valid;
  int teacher_ctas;
  const float* entropy;
  const int* state;
  const int* ids;
  const float* probs;
  float* loss_rows;
  unsigned* ticket;
  float* loss;
  int* err;
  int list;
  int n_cols;
  int64_t n_rows;
  float temperature, inv_t, hard_weight, loss_scale;
};

// Rows that count, at least 1 (all threads return the same number).
__device__ __forceinline__ float count_valid(const RowArgs& a) {
  int n = 0;
  for (int i = 0; i < a.teacher_ctas; ++i) n += a.valid[i].x;
  return (float)(n < 1 ? 1 : n);
}

// The CTA that ends last adds the row losses up in a fixed order.
__device__ __forceinline__ void finish_loss(const RowArgs& a, float n) {
  __shared__ bool last;
  __shared__ double red[32];
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < a.n_rows; i += blockDim.x) s += (double)__ldcg(a.loss_rows + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
    *a.loss = (float)(s / (double)n);
    int bad = 0;
    for (int i = 0; i < a.teacher_ctas; ++i) bad |= a.valid[i].y;
    *a.err = bad != 0;
  }
}

// One CTA per row, element loops (any stride and alignment).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_rows_generic(
    const T* logits, int64_t lstride, T* grad, int64_t gstride, RowArgs a) {
  __shared__ float red[32];
  __shared__ float picked[kMaxSlots + 1];
  const float n = count_valid(a);
  const bool two = a.temperature != 1.0f;
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    const T* src = logits + row * lstride;
    T* dst = grad ? grad + row * gstride : nullptr;
    const int state = a.state[row];
    if (state == kSkip || state == kBad) {
      const float z = state == kBad ? __int_as_float(0x7fc00000) : 0.f;
      if (threadIdx.x == 0) a.loss_rows[row] = z;
      if (dst)
        for (int c = threadIdx.x; c < a.n_cols; c += blockDim.x) dst[c] = Elt<T>::from_f(z);
      continue;
    }
    const int* ids = a.ids + row * a.list;
    const float* probs = a.probs + row * a.list;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < a.n_cols; c += blockDim.x) m = fmaxf(m, Elt<T>::to_f(src[c]));
    m = block_max(m, red);
    const float base = m == -INFINITY ? 0.f : m;
    float zt = 0.f, z1 = 0.f, dot = 0.f;
    for (int c = threadIdx.x; c < a.n_cols; c += blockDim.x) {
      const float d = Elt<T>::to_f(src[c]) - base;
      zt += expf(d * a.inv_t);
      if (two) z1 += expf(d);
    }
    for (int j = threadIdx.x; j < a.list; j += blockDim.x) {
      const int c = ids[j];
      const float v = c >= 0 ? Elt<T>::to_f(src[c]) - base : 0.f;
      picked[j] = v;
      if (c >= 0 && probs[j] != 0.f) dot = fmaf(probs[j], v, dot);
    }
    zt = block_sum(zt, red);
    z1 = two ? block_sum(z1, red) : zt;
    dot = block_sum(dot, red);
    const float hw = (state & kHard) ? a.hard_weight : 0.f;
    const float sw = (state & kSoft) ? 1.f - a.hard_weight : 0.f;
    if (threadIdx.x == 0) {  // a part of weight 0 is left out, even where it is infinite
      float l = 0.f;
      if (sw > 0.f)
        l = sw * a.temperature * a.temperature * (a.entropy[row] - dot * a.inv_t + logf(zt));
      if (hw > 0.f) l += hw * (logf(z1) - picked[a.list - 1]);
      a.loss_rows[row] = l;
    }
    if (dst) {
      const float ct = sw * a.temperature * a.loss_scale / n, c1 = hw * a.loss_scale / n;
      const float kt = ct / zt, k1 = c1 / z1;
      auto dense = [&](float d) {
        float g = kt * expf(d * a.inv_t);
        if (two) g = fmaf(k1, expf(d), g);
        else g = fmaf(k1, expf(d * a.inv_t), g);
        return g;
      };
      for (int c = threadIdx.x; c < a.n_cols; c += blockDim.x)
        dst[c] = Elt<T>::from_f(dense(Elt<T>::to_f(src[c]) - base));
      __syncthreads();  // the listed places are written over the dense values
      for (int j = threadIdx.x; j < a.list; j += blockDim.x) {
        const int c = ids[j];
        if (c >= 0)
          dst[c] = Elt<T>::from_f(dense(picked[j]) - ct * probs[j] -
                                  ((state & kHard) && j == a.list - 1 ? c1 : 0.f));
      }
    }
    __syncthreads();  // picked is the next row's from here
  }
  finish_loss(a, n);
}

template <typename T>
int rows_t(const void* logits, int64_t ls, void* grad, int64_t gs, const RowArgs& a,
           cudaStream_t st) {
  const int64_t most = (int64_t)num_sms() * kRowCtasPerSm;
  const int grid = (int)(a.n_rows < most ? a.n_rows : most);
  distill_rows_generic<T><<<grid < 1 ? 1 : grid, kRowThreads, 0, st>>>(
      static_cast<const T*>(logits), ls, static_cast<T*>(grad), gs, a);
  return launch_status("fk_distill(rows)");
}

template <typename T>
int teacher_t(const int64_t* idx, const void* top, int k, const int64_t* targets,
              int64_t ignore_index, int64_t n_rows, int64_t n_cols, float inv_t,
              const Workspace& ws, int* ctas, cudaStream_t st) {
  int table = 32;
  while (table < 2 * k) table *= 2;
  const int smem = kTeacherWarps * (2 * k + table) * 4;
  const int64_t want = (n_rows + kTeacherWarps - 1) / kTeacherWarps;
  *ctas = (int)(want < 1 ? 1 : want > kTeacherCtas ? kTeacherCtas : want);
  auto kern = distill_teacher<T>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<*ctas, kTeacherWarps * 32, smem, st>>>(idx, static_cast<const T*>(top), k, table, targets,
                                                ignore_index, n_rows, n_cols, inv_t, ws);
  return launch_status("fk_distill(teacher)");
}

}  // namespace
}  // namespace fk

extern "C" int fk_distill_workspace_size(int64_t n_rows, int k, size_t* bytes) {
  FK_CHECK_ARG(bytes != nullptr, "fk_distill_workspace_size: null output");
  FK_CHECK_ARG(n_rows >= 0 && k >= 1, "fk_distill_workspace_size: bad shape");
  fk::Workspace w;
  *bytes = fk::ws_layout(nullptr, n_rows, k, &w);
  return FK_OK;
}

extern "C" int fk_distill(const void* logits, int64_t row_stride, void* grad,
                          int64_t grad_row_stride, const int64_t* teacher_idx,
                          const void* teacher_logits, int teacher_dtype, int k,
                          const int64_t* targets, int64_t n_rows, int64_t n_cols,
                          int64_t ignore_index, float temperature, float hard_weight,
                          float loss_scale, int dtype, float* loss, int* err_flag,
                          void* workspace, size_t workspace_bytes, void* stream) {
  FK_CHECK_ARG(n_rows >= 0 && n_cols >= 1 && k >= 1, "fk_distill: bad shape");
  FK_CHECK_ARG(n_cols < ((int64_t)1 << 31) - 4096, "fk_distill: n_cols too large");
  if (k > fk::kMaxSlots)
    return fk::fail(FK_ERR_UNSUPPORTED, "fk_distill: k=%d exceeds %d", k, fk::kMaxSlots);
  FK_CHECK_ARG(fk::valid_dtype(dtype) && fk::valid_dtype(teacher_dtype), "fk_distill: bad dtype");
  FK_CHECK_ARG(row_stride >= n_cols && (!grad || grad_row_stride >= n_cols),
               "fk_distill: stride < n_cols");
  FK_CHECK_ARG(temperature > 0.f && temperature < INFINITY, "fk_distill: temperature must be > 0");
  FK_CHECK_ARG(hard_weight >= 0.f && hard_weight <= 1.f, "fk_distill: hard_weight outside [0, 1]");
  FK_CHECK_ARG(loss && err_flag, "fk_distill: null pointer");
  FK_CHECK_ARG(n_rows == 0 || (logits && teacher_idx && teacher_logits),
               "fk_distill: null pointer");
  fk::Workspace ws;
  const size_t need = fk::ws_layout(workspace, n_rows, k, &ws);
  if (workspace == nullptr || workspace_bytes < need || !fk::aligned16(workspace))
    return fk::fail(FK_ERR_WORKSPACE, "fk_distill: need %zu aligned workspace bytes, got %zu",
                    need, workspace_bytes);
  cudaStream_t st = fk::as_stream(stream);
  int ctas = 0, s = FK_OK;
  FK_DISPATCH_DTYPE(teacher_dtype,
                    s = fk::teacher_t<scalar_t>(teacher_idx, teacher_logits, k, targets,
                                                ignore_index, n_rows, n_cols, 1.0f / temperature,
                                                ws, &ctas, st));
  if (s != FK_OK) return s;
  fk::RowArgs a;
  a.valid = ws.valid;
  a.teacher_ctas = ctas;
  a.entropy = ws.entropy;
  a.state = ws.state;
  a.ids = ws.ids;
  a.probs = ws.probs;
  a.loss_rows = ws.loss_rows;
  a.ticket = ws.ticket;
  a.loss = loss;
  a.err = err_flag;
  a.list = k + 1;
  a.n_cols = (int)n_cols;
  a.n_rows = n_rows;
  a.temperature = temperature;
  a.inv_t = 1.0f / temperature;
  a.hard_weight = targets ? hard_weight : 0.f;
  a.loss_scale = loss_scale;
  FK_DISPATCH_DTYPE(dtype, s = fk::rows_t<scalar_t>(logits, row_stride, grad, grad_row_stride, a,
                                                    st));
  return s;
}
