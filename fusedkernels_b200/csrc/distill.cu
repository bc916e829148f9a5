// Distillation from a teacher's top logits, optionally mixed with the hard label: loss and
// gradient.  Per row, over the used slots j (id i_j >= 0, teacher logit t_j):
//
//   p = softmax(t / T) over the slots,  q = softmax(s / T) over the vocabulary
//   soft = T^2 * sum_j p_j (log p_j - s_{i_j}/T + lse(s/T)),  hard = lse(s) - s_y
//   loss = 1/n * sum_rows [(1-a) soft + a hard]
//   dloss/ds_c = 1/n * [(1-a) T (q_c - P_c) + a (softmax(s)_c - [c = y])],
//   P_c = sum of the p_j whose id is c.
//
// The teacher's side of a row is small and is done first, by a few lanes per row: it leaves a
// list of (id, P) with every id once and the label's entry last, the row's sum p log p, and
// partial counts of the rows that count (n).  The second kernel then needs every logit once
// for the two sums and once for its gradient, and the gradient at the listed ids is computed
// from the logit itself, in 32 bits, and rounded once.
#include "common.cuh"
#include "exp.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace fk {
namespace {

constexpr int kMaxSlots = 1024;
constexpr int kTeacherWarps = 8;
constexpr int kTeacherCtas = 1024;  // partial counts that every CTA of the second kernel adds up
constexpr int kMaxRowCtasPerSm = 16;
// Row states.
constexpr int kSkip = 0, kSoft = 1, kHard = 2, kBad = 4;

struct Workspace {
  int2* valid;       // [kTeacherCtas] (rows that count, rows with an id out of range)
  unsigned* ticket;
  double* sums;      // [kMaxRowCtasPerSm * SMs]  loss of the rows of one CTA
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
  w->sums = reinterpret_cast<double*>(take((size_t)num_sms() * kMaxRowCtasPerSm * 8));
  w->entropy = reinterpret_cast<float*>(take(n * 4));
  w->state = reinterpret_cast<int*>(take(n * 4));
  w->ids = reinterpret_cast<int*>(take(n * list * 4));
  w->probs = reinterpret_cast<float*>(take(n * list * 4));
  return at;
}

// ------------------------------------------------------------------ teacher -------------
// Shared-memory words of a row; the rows of a warp lie 8 banks apart.
__host__ __device__ inline int row_ints(int k, int log_table) {
  return (2 * k + (1 << log_table) + 31) / 32 * 32 + 8;
}

// G lanes of a warp take a row.  Shared memory per row: ids[k], p[k], and a table that finds
// ids standing twice: every slot writes its number at its id's hash and reads back whose number
// is there.  Its own: the id is settled.  A slot of the same id: it stands twice.  Another id's:
// the slot goes on to the next round, with another hash.  Slots of one id stay together until
// one of them is settled and the others see it.  (Plain stores: inserting by atomicCAS took
// 3.7 clocks a slot on an SM, 14 of the 18 us at 8192 rows of 64.)
template <typename T, int G>
__global__ void __launch_bounds__(kTeacherWarps * 32) distill_teacher(
    const int64_t* __restrict__ idx, const T* __restrict__ top, int k, int log_table,
    const int64_t* __restrict__ targets, int64_t ignore_index, int n_rows, int64_t n_cols,
    float inv_t, Workspace ws) {
  extern __shared__ int smem[];
  __shared__ int valid_rows, bad_rows;
  constexpr int kRows = kTeacherWarps * 32 / G;  // of a CTA at a time
  const int at = threadIdx.x % G, slot = threadIdx.x / G;
  int* ids = smem + slot * row_ints(k, log_table);
  float* p = reinterpret_cast<float*>(ids + k);
  int* table = ids + 2 * k;
  auto group_max = [](float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  auto group_sum = [](float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto group_any = [&](bool b) {
    const unsigned all = __ballot_sync(0xffffffffu, b);
    const unsigned mine = (G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << (threadIdx.x & 31 & ~(G - 1)));
    return (all & mine) != 0;
  };
  ptx::let_next_kernel_start();
  if (threadIdx.x == 0) {
    valid_rows = bad_rows = 0;
    if (blockIdx.x == 0) *ws.ticket = 0;
  }
  __syncthreads();
  const int list = k + 1;
  for (int base = blockIdx.x * kRows; base < n_rows; base += gridDim.x * kRows) {
    const bool there = base + slot < n_rows;
    const int row = there ? base + slot : n_rows - 1;  // idle groups go along on the last row
    const int64_t* row_idx = idx + (int64_t)row * k;
    const T* row_top = top + (int64_t)row * k;
    const int64_t y = targets ? targets[row] : -1;
    const bool ignored = targets && y == ignore_index;
    bool bad = targets && !ignored && (y < 0 || y >= n_cols);
    float m = -INFINITY;
    bool twice = false, nan = false;
#pragma unroll 4
    for (int j = at; j < k; j += G) {
      const int64_t id = row_idx[j];
      const float v = Elt<T>::to_f(row_top[j]);
      const bool out = id >= n_cols;
      bad = bad || (out && !ignored);
      const int c = (id < 0 || out) ? -1 : (int)id;
      ids[j] = c;
      p[j] = v;
      if (c >= 0) {
        m = fmaxf(m, v);
        nan = nan || v != v;
      }
    }
    m = group_max(m);
    nan = group_any(nan);  // (votes are for the whole warp: never behind a row's condition)
    bad = group_any(bad);
    const bool held = m != -INFINITY || nan;
    __syncwarp();
    float z = 0.f;
    unsigned open = 0;  // this lane's slots that are not settled
    for (int j = at, i = 0; j < k; j += G, ++i) {
      if (ids[j] >= 0 && held) {
        z += expf((p[j] - m) * inv_t);
        open |= 1u << i;
      } else {
        ids[j] = -1;
      }
    }
    for (unsigned round = 0; __any_sync(0xffffffffu, open != 0); ++round) {
      const unsigned factor = 2654435761u + round * 1640531526u;  // odd
      for (unsigned o = open; o; o &= o - 1) {
        const int j = at + (__ffs(o) - 1) * G;
        table[(unsigned)ids[j] * factor >> (32 - log_table)] = j;
      }
      __syncwarp();
      for (unsigned o = open; o; o &= o - 1) {
        const int i = __ffs(o) - 1, j = at + i * G, c = ids[j];
        const int there_j = table[(unsigned)c * factor >> (32 - log_table)];
        const bool same = ids[there_j] == c;
        if (same) open &= ~(1u << i);
        twice = twice || (same && there_j != j);
      }
      __syncwarp();
    }
    twice = group_any(twice);
    z = group_sum(z);
    const float lz = logf(z), inv_z = held ? 1.0f / z : 0.f;
    float ent = 0.f;
    for (int j = at; j < k; j += G) {
      float pj = 0.f;
      if (ids[j] >= 0) {
        const float d = (p[j] - m) * inv_t;
        pj = expf(d) * inv_z;
        if (pj > 0.f) ent = fmaf(pj, d - lz, ent);
        else if (pj != pj) ent = pj;
      }
      p[j] = pj;
    }
    ent = group_sum(ent);
    __syncwarp();
    int state = kSkip;
    if (!ignored && bad) state = kBad;
    else if (!ignored) state = (held ? kSoft : 0) | (targets ? kHard : 0);
    const int label = (state & kHard) ? (int)y : -1;
    // The list: every id once, at its first slot, with the sum of its probabilities; the
    // label's at the end.
    float py = 0.f;
    int* out_ids = ws.ids + (int64_t)row * list;
    float* out_probs = ws.probs + (int64_t)row * list;
    for (int j = at; j < k; j += G) {
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
      if (c >= 0 && c == label) {
        py += pj;
        c = -1;
      }
      if (there) {
        out_ids[j] = c;
        out_probs[j] = c >= 0 ? pj : 0.f;
      }
    }
    py = group_sum(py);
    if (at == 0 && there) {
      out_ids[k] = label;
      out_probs[k] = py;
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
  double* sums;
  unsigned* ticket;
  float* loss;
  int* err;
  int list;
  int n_cols;
  int64_t n_rows;
  float temperature, inv_t, hard_weight, loss_scale;
  float inv_p;   // kPowers: 1 / P
  bool q2, p4;   // Q = 2, P = 4 (else 1, 3)
};

// Rows that count, at least 1 (whole warps call; all threads return the same number).
__device__ __forceinline__ float count_valid(const RowArgs& a) {
  int n = 0;
  for (int i = threadIdx.x & 31; i < a.teacher_ctas; i += 32) n += a.valid[i].x;
  n = __reduce_add_sync(0xffffffffu, n);
  return (float)(n < 1 ? 1 : n);
}

// Sum over the CTA's threads in a fixed order (valid in thread 0).
__device__ __forceinline__ double block_total(double s) {
  __shared__ double red[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
  return s;
}

// Every thread brings its part of the loss of the CTA's rows; the CTA that ends last adds the
// CTAs' sums up in a fixed order (at most 16 per SM).
__device__ __forceinline__ void finish_loss(const RowArgs& a, double mine) {
  __shared__ bool last;
  mine = block_total(mine);
  if (threadIdx.x == 0) {
    a.sums[blockIdx.x] = mine;
    __threadfence();
    last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += blockDim.x) s += __ldcg(a.sums + i);
  s = block_total(s);
  int bad = 0;
  for (int i = threadIdx.x; i < a.teacher_ctas; i += blockDim.x) bad |= a.valid[i].y;
  bad = __syncthreads_or(bad);
  const float n = count_valid(a);
  if (threadIdx.x == 0) {
    *a.loss = (float)(s / (double)n);
    *a.err = bad != 0;
  }
}

// ------------------------------------------------------------------ rows, any layout ----
constexpr int kGenericThreads = 256;

// One CTA per row, element loops (any stride, alignment and length).  Three passes over the row:
// 3.1 ms at 2048 x 262144 bf16 for 0.33 of bytes, 0.97 ms at 1024 x 151936 fp32 for 0.19.
template <typename T>
__global__ void __launch_bounds__(kGenericThreads) distill_rows_generic(
    const T* logits, int64_t lstride, T* grad, int64_t gstride, RowArgs a) {
  __shared__ float red[32];
  __shared__ float picked[kMaxSlots + 1];
  const float n = count_valid(a);
  const bool two = a.temperature != 1.0f;
  double total = 0.0;
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    const T* src = logits + row * lstride;
    T* dst = grad ? grad + row * gstride : nullptr;
    const int state = a.state[row];
    if (state == kSkip || state == kBad) {
      const float z = state == kBad ? __int_as_float(0x7fc00000) : 0.f;
      if (threadIdx.x == 0) total += (double)z;
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
      total += (double)l;
    }
    if (dst) {
      const float ct = sw * a.temperature * a.loss_scale / n, c1 = hw * a.loss_scale / n;
      const float kt = ct / zt, k1 = c1 / z1;
      auto dense = [&](float d) {
        const float e = expf(d * a.inv_t);
        return fmaf(kt, e, k1 * (two ? expf(d) : e));
      };
      for (int c = threadIdx.x; c < a.n_cols; c += blockDim.x)
        dst[c] = Elt<T>::from_f(dense(Elt<T>::to_f(src[c]) - base));
      __syncthreads();  // the listed places are written over the dense values
      for (int j = threadIdx.x; j < a.list; j += blockDim.x) {
        const int c = ids[j];
        if (c >= 0)
          dst[c] = Elt<T>::from_f(dense(picked[j]) - (sw > 0.f ? ct * probs[j] : 0.f) -
                                  ((state & kHard) && j == a.list - 1 ? c1 : 0.f));
      }
    }
    __syncthreads();  // picked is the next row's from here
  }
  finish_loss(a, total);
}

// ------------------------------------------------------------------ rows, 16-byte packets
// A cluster of 1, 2, 4 or 8 CTAs takes a row; each CTA has a slice of its 16-byte packets, at
// most KP per thread.  A slice arrives in a shared-memory buffer by cp.async.bulk, moves to
// registers, and its buffer is refilled with the next row's as soon as every thread has taken
// its packets: the next row is on its way while this one is worked on.
//
// A thread forms the sum of exp((x - m_t) / T) with its own maximum m_t; the CTAs of a row
// exchange (m, z) by st.async into each other's shared memory.  16-bit packets stay in
// registers and the gradient's exponentials are formed anew: keeping the first ones in 32 bits
// takes twice the registers, half as many rows are then in flight, and their latency shows
// (810 against 717 us at 8192 x 128256 bf16, before x - max was formed; 725 since).  32-bit packets
// give their registers to their exponentials, which the gradient only scales.
//
// Elements before the first and after the last 16-byte boundary of a row (any odd width or
// offset) are taken singly by the first CTA.  Logits and gradient have to have the same
// offset from a 16-byte boundary in every row; other layouts take the generic kernel.
constexpr int kMaxStages = 3;
constexpr uint32_t kPolls = 1u << 21;  // of a wait, before it gives up

// exp(d) of a scaled difference d <= 0: 16-bit gradients round to 8 or 11 bits, so one ex2 is
// exact enough; 32-bit ones take expf.
template <typename T>
__device__ __forceinline__ float exp_of(float d) { return ex2f(d * kLog2e); }
template <>
__device__ __forceinline__ float exp_of<float>(float d) { return expf(d); }

template <typename T> struct Pair;  // two neighbouring elements
template <> struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  __nv_bfloat162 v;
  __device__ __forceinline__ float2 f() const { return __bfloat1622float2(v); }
  __device__ __forceinline__ void set(float2 a) { v = __float22bfloat162_rn(a); }
  __device__ __forceinline__ void take_max(const Pair& b) { v = __hmax2(v, b.v); }
};
template <> struct Pair<__half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  __half2 v;
  __device__ __forceinline__ float2 f() const { return __half22float2(v); }
  __device__ __forceinline__ void set(float2 a) { v = __float22half2_rn(a); }
  __device__ __forceinline__ void take_max(const Pair& b) { v = __hmax2(v, b.v); }
};
template <> struct Pair<float> {
  static constexpr uint32_t kNegInf = 0xff800000u;
  float2 v;
  __device__ __forceinline__ float2 f() const { return v; }
  __device__ __forceinline__ void set(float2 a) { v = a; }
  __device__ __forceinline__ void take_max(const Pair& b) {
    v = make_float2(fmaxf(v.x, b.v.x), fmaxf(v.y, b.v.y));
  }
};
// A 16-byte packet as pairs.
template <typename T>
union PairPacket {
  static constexpr int N = 16 / sizeof(Pair<T>);
  uint4 u;
  Pair<T> p[N];
  __device__ __forceinline__ PairPacket() {}
};

// What a row needs: softmax at one temperature, or at two (the soft part's, T, and 1).  Where T is
// a ratio of small numbers P / Q, one exponential b = exp(d / P) gives both: b^Q = exp(d / T) and
// b^P = exp(d), with Q and P times b's relative error (2 to 3 ulp).  kSquare is T = 2, kPowers T =
// 3, 4 and 3 / 2.  At 8192 x 128256 bf16 (651 us of bytes): one temperature 725 us, T = 2 749,
// kPowers 950, two exponentials per logit (T = 2.5) 1451: the ex2 unit alone takes 900 for them,
// and 280 bytes are spilled.  At 2048 x 50257 fp32 (128 us of bytes): T = 2 149, T = 3 228, T =
// 2.5 285.
enum Mode { kOne, kTwo, kSquare, kPowers };

// (maximum, sum exp((x - max) / T), sum exp(x - max)) of a set of logits.
struct Stat {
  float m, z, z1;
};
// Joins the sets of the lanes; WIDTH of them differ (lane l holds set l % WIDTH).
template <typename T, Mode M, int WIDTH>
__device__ __forceinline__ Stat join(Stat s, float inv_t) {
  Stat r;
  r.m = warp_redux_max(s.m);
  const float d = s.m == -INFINITY ? 0.f : s.m - r.m;  // an empty set's sum is 0, or NaN
  r.z = s.z * exp_of<T>(d * inv_t);
  r.z1 = M != kOne ? s.z1 * exp_of<T>(d) : 0.f;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
    if (M != kOne) r.z1 += __shfl_xor_sync(0xffffffffu, r.z1, o);
  }
  return r;
}

template <typename T, Mode M, bool KEEP, int THREADS, int KP, int MIN_CTAS>
__global__ void __launch_bounds__(THREADS, MIN_CTAS) distill_rows(
    const T* logits, int64_t lstride, T* grad, int64_t gstride, int stage_bytes, int stages,
    int log_c, RowArgs a) {
  using PK = PairPacket<T>;
  constexpr int VN = 16 / (int)sizeof(T);
  constexpr int NP = PK::N;
  constexpr int kWarps = THREADS / 32;
  extern __shared__ __align__(128) unsigned char ring[];
  float* picked = reinterpret_cast<float*>(ring + stages * stage_bytes);  // [list]
  __shared__ __align__(8) uint64_t full[kMaxStages];
  __shared__ __align__(8) uint64_t xbar[2];
  __shared__ __align__(16) float4 xch[2][8];
  __shared__ Stat wred[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = 1 << log_c, rank = (int)ptx::cluster_ctarank();
  const int n_rows = (int)a.n_rows, first = (int)(blockIdx.x >> log_c);
  const int step = (int)(gridDim.x >> log_c);
  const bool loader = tid == THREADS - 32;  // the last warp's first lane starts the loads

  // A row's 16-byte packets and this CTA's share of them.
  struct Slice {
    int head, packets, start, count;
  };
  auto slice_of = [&](const T* src) {
    Slice s;
    s.head = (int)((0u - (unsigned)reinterpret_cast<uintptr_t>(src)) & 15u) / (int)sizeof(T);
    if (s.head > a.n_cols) s.head = a.n_cols;
    s.packets = (int)((unsigned)(a.n_cols - s.head) / (unsigned)VN);
    const int per = (s.packets + C - 1) >> log_c;
    s.start = rank * per;
    const int left = s.packets - s.start;
    s.count = left < per ? (left < 0 ? 0 : left) : per;
    return s;
  };
  auto issue = [&](int row, int q) {  // loader: this CTA's slice of a row into stage q
    if (row >= n_rows) return;
    const T* src = logits + row * lstride;
    const Slice s = slice_of(src);
    ptx::fence_proxy_async_smem();
    if (s.count > 0) {
      ptx::mbar_arrive_expect_tx(&full[q], (uint32_t)s.count * 16u);
      ptx::bulk_g2s(ring + q * stage_bytes, src + s.head + s.start * VN, (uint32_t)s.count * 16u,
                    &full[q]);
    } else {
      ptx::mbar_arrive(&full[q]);
    }
  };
  if (tid == 0) {
    for (int q = 0; q < stages; ++q) ptx::mbar_init(&full[q], 1);
    ptx::mbar_init(&xbar[0], 1);
    ptx::mbar_init(&xbar[1], 1);
    ptx::fence_mbar_init();
  }
  if (C > 1) ptx::cluster_sync();
  else __syncthreads();
  if (loader)
    for (int q = 0; q < stages; ++q) issue(first + q * step, q);

  ptx::wait_for_previous_kernel();  // the logits are older; the rest is the teacher kernel's
  const float inv_n = 1.0f / count_valid(a);
  const float inv_t = a.inv_t;
  const float inv_b = M == kPowers ? a.inv_p : inv_t;  // b = exp(d * inv_b)
  const float ct_row = inv_b * kLog2e;                  // exponent of 2 per unit of logit
  auto powers = [&](float b, float& f, float& f1) {
    const float b2 = b * b;
    f = a.q2 ? b2 : b;
    f1 = b2 * (a.p4 ? b2 : b);
  };
  auto powers_of_pair = [&](float2 b, float2& f, float2& f1) {
    const float2 b2 = __fmul2_rn(b, b);
    f = a.q2 ? b2 : b;
    f1 = __fmul2_rn(b2, a.p4 ? b2 : b);
  };
  const bool same_slice = lstride % VN == 0;  // every row has the first row's offset
  const bool lists = warp * 32 < a.list;      // this warp has listed elements to handle
  bool ok = true;
  double total = 0.0;
  int q = 0, phase = 0, xb = 0, xphase = 0;
  // What the row brings besides its logits is read one row ahead.
  const int* next_id = a.ids + (int64_t)first * a.list + tid;
  const float* next_p = a.probs + (int64_t)first * a.list + tid;
  int state = 0, my_id = -1;
  float my_p = 0.f, entropy = 0.f;
  auto read_ahead = [&](int row) {
    if (row >= n_rows) return;
    state = a.state[row];
    if (tid == THREADS - 1) entropy = a.entropy[row];
    if (lists) {
      if (tid < a.list) {
        my_id = *next_id;
        my_p = *next_p;
      }
      next_id += (int64_t)step * a.list;
      next_p += (int64_t)step * a.list;
    }
  };
  read_ahead(first);
  const T* src = logits + first * lstride;
  T* dst = grad + first * gstride;
  Slice sl = slice_of(src);
  for (int row = first; row < n_rows; row += step) {
    const int row_state = state, id = my_id;
    const float p_id = my_p, row_entropy = entropy;
    float xs = -INFINITY;  // an element outside the packets
    int xs_at = -1;
    if (rank == 0 && warp < 2) {
      const int tail = sl.head + sl.packets * VN;
      if (tid < sl.head) xs_at = tid;
      else if (tid >= 32 && tid - 32 < a.n_cols - tail) xs_at = tail + tid - 32;
      if (xs_at >= 0) xs = Elt<T>::to_f(src[xs_at]);
    }
    ok = ptx::mbar_wait(&full[q], (uint32_t)phase, ok ? kPolls : 1u) && ok;
    const unsigned char* stage = ring + q * stage_bytes;
    PK p[KP];
    // All but the last packet of every thread are there as a rule (one branch for the row).
    const bool most_full = M != kTwo && (KP - 1) * THREADS <= sl.count;
    const uint4* at = reinterpret_cast<const uint4*>(stage) + tid;
    constexpr uint32_t w = Pair<T>::kNegInf;
    if (most_full) {
#pragma unroll
      for (int u = 0; u + 1 < KP; ++u) p[u].u = at[u * THREADS];
      p[KP - 1].u = make_uint4(w, w, w, w);
      if (tid + (KP - 1) * THREADS < sl.count) p[KP - 1].u = at[(KP - 1) * THREADS];
    } else {
#pragma unroll
      for (int u = 0; u < KP; ++u) {
        p[u].u = make_uint4(w, w, w, w);
        if (tid + u * THREADS < sl.count) p[u].u = at[u * THREADS];
      }
    }
    // Listed elements of this slice: the same thread handles a listed place all through.
    auto mine = [&](int c) {  // whether element c is this CTA's
      const unsigned off = (unsigned)(c - sl.head);
      if (c < 0) return false;
      if (off >= (unsigned)(sl.packets * VN)) return rank == 0;
      return off / VN - (unsigned)sl.start < (unsigned)sl.count;
    };
    auto value = [&](int c) {  // its logit
      const unsigned off = (unsigned)(c - sl.head);
      if (off >= (unsigned)(sl.packets * VN)) return Elt<T>::to_f(src[c]);
      return Elt<T>::to_f(reinterpret_cast<const T*>(stage)[(int)off - sl.start * VN]);
    };
    bool has = false;
    float x_id = 0.f;
    if (lists) {
      has = mine(id);
      if (has) x_id = value(id);
      for (int j = tid + THREADS; j < a.list; j += THREADS) {
        const int c = a.ids[(int64_t)row * a.list + j];
        if (mine(c)) picked[j] = value(c);
      }
    }
    // This thread's maximum and exponentials.
    float my_m;
    {
      Pair<T> top = p[0].p[0];
#pragma unroll
      for (int k = 1; k < KP * NP; ++k) top.take_max(p[k / NP].p[k % NP]);
      const float2 f = top.f();
      my_m = fmaxf(fmaxf(f.x, f.y), xs);
    }
    const float base = my_m == -INFINITY ? 0.f : my_m;
    // The maximum goes off first: folded into the exponent as the constant -max log2(e) / T it
    // would leave that product's rounding in every term, and overflow at a mask of the type's
    // lowest value.
    auto exp_one = [&](float x, float& f, float& f1) {
      const float d = x - base;
      if constexpr (sizeof(T) == 2) {
        f = ex2f(d * ct_row);
        if constexpr (M == kTwo) f1 = ex2f(d * kLog2e);
      } else {
        f = exp2_of(d * inv_b);
        if constexpr (M == kTwo) f1 = exp2_of(d);
      }
      if constexpr (M == kSquare) f1 = f * f;
    };
    float2 e[KEEP ? KP : 1][NP], e1[KEEP && M == kTwo ? KP : 1][NP];
    float2 z = make_float2(0.f, 0.f), z1 = z;
    if (xs_at >= 0) {
      exp_one(xs, z.x, z1.x);
      if constexpr (M == kPowers) powers(z.x, z.x, z1.x);
    }
#pragma unroll
    for (int u = 0; u < KP; ++u)
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const float2 x = p[u].p[k].f();
        float2 f, f1 = make_float2(0.f, 0.f);
        if constexpr (sizeof(T) == 2 && M != kTwo) {
          const float2 t = __fmul2_rn(__fadd2_rn(x, make_float2(-base, -base)),
                                      make_float2(ct_row, ct_row));
          f = make_float2(ex2f(t.x), ex2f(t.y));
          if constexpr (M == kPowers) {
            float2 g;
            powers_of_pair(f, g, f1);
            z = __fadd2_rn(z, g);
            z1 = __fadd2_rn(z1, f1);
          } else {
            z = __fadd2_rn(z, f);
            if constexpr (M == kSquare) z1 = __ffma2_rn(f, f, z1);
          }
        } else {
          exp_one(x.x, f.x, f1.x);
          exp_one(x.y, f.y, f1.y);
          float2 g = f;
          if constexpr (M == kPowers) {
            powers(f.x, g.x, f1.x);
            powers(f.y, g.y, f1.y);
          }
          z.x += g.x;
          z.y += g.y;
          if constexpr (M != kOne) {
            z1.x += f1.x;
            z1.y += f1.y;
          }
        }
        if constexpr (KEEP) {
          e[u][k] = f;
          if constexpr (M == kTwo) e1[u][k] = f1;
        }
      }
    // (A thread whose wait ran out poisons the row's sums for all of them.)
    if (!ok) z.x = __int_as_float(0x7fc00000);
    Stat st = join<T, M, 32>(Stat{my_m, z.x + z.y, M != kOne ? z1.x + z1.y : 0.f}, inv_t);
    if (lane == 0) wred[warp] = st;
    __syncthreads();  // the stage has been read by all
    if (loader && ok) issue(row + stages * step, q);
    if (C == 1 || warp == 0) st = join<T, M, kWarps>(wred[lane & (kWarps - 1)], inv_t);
    if (C > 1) {
      if (warp == 0) {
        if (lane == 0) ptx::mbar_arrive_expect_tx(&xbar[xb], (uint32_t)C * 16u);
        if (lane < C)
          ptx::st_async16(ptx::peer_smem(&xch[xb][rank], (uint32_t)lane),
                          make_float4(st.m, st.z, st.z1, 0.f),
                          ptx::peer_smem(&xbar[xb], (uint32_t)lane));
        __syncwarp();
      }
      read_ahead(row + step);
      ok = ptx::mbar_wait(&xbar[xb], (uint32_t)xphase, ok ? kPolls : 1u) && ok;
      const float4 f = xch[xb][lane & (C - 1)];
      const bool copy = (lane & 7) >= C;  // of a smaller cluster: counted once
      st = join<T, M, 8>(Stat{f.x, copy ? 0.f : f.y, copy ? 0.f : f.z}, inv_t);
    } else {
      read_ahead(row + step);
    }
    if (!ok) st.z = st.z1 = __int_as_float(0x7fc00000);  // (or the wait for the other CTAs)
    const float hw = (row_state & kHard) ? a.hard_weight : 0.f;
    const float sw = (row_state & kSoft) ? 1.f - a.hard_weight : 0.f;
    const float ct = sw * a.temperature * a.loss_scale * inv_n, c1 = hw * a.loss_scale * inv_n;
    // (2 ulp, as the exponentials they meet.  A full division and log2f keep more registers and
    // spill: T = 2 842 against 816 us at 8192 x 128256 bf16, fp16 247 against 237 at 8192 x 32000.)
    const float kt = __fdividef(M != kOne ? ct : ct + c1, st.z);
    const float k1 = M != kOne ? __fdividef(c1, st.z1) : 0.f;
    const bool plain = row_state == kSkip || row_state == kBad;
    const float fill = row_state == kBad || !ok ? __int_as_float(0x7fc00000) : 0.f;

    if (grad) {
      uint4* out = reinterpret_cast<uint4*>(dst + sl.head + sl.start * VN) + tid;
      if (plain) {
        PK o;
#pragma unroll
        for (int k = 0; k < NP; ++k) o.p[k].set(make_float2(fill, fill));
        for (int v = tid; v < sl.count; v += THREADS, out += THREADS) __stcs(out, o.u);
        if (xs_at >= 0) dst[xs_at] = Elt<T>::from_f(fill);
      } else {
        // 16 bits: the factor k / z goes into the exponent.
        const float ot = __log2f(kt), o1 = __log2f(k1);
        // wt exp(d / T) and, where one exponential gives both, + w1 exp(d).
        auto both = [&](float b, float wt, float w1) {
          if constexpr (M == kPowers) {
            float f, f1;
            powers(b, f, f1);
            return fmaf(f1, w1, f * wt);
          }
          return b * (M == kSquare ? fmaf(b, w1, wt) : wt);
        };
        auto dense = [&](float x) {
          const float d = x - st.m;
          float g;
          if constexpr (sizeof(T) == 2) {
            if constexpr (M == kSquare || M == kPowers) {
              g = both(ex2f(d * ct_row), kt, k1);
            } else {
              g = ex2f(fmaf(d, ct_row, ot));
              if constexpr (M == kTwo) g += ex2f(fmaf(d, kLog2e, o1));
            }
          } else {
            g = both(exp2_of(d * inv_b), kt, k1);
            if constexpr (M == kTwo) g = fmaf(exp2_of(d), k1, g);
          }
          return g;
        };
        const bool none = my_m == -INFINITY;
        // (A thread with nothing but -inf: 0, or NaN where the row's sum is.)
        const float ft = KEEP ? (none ? 0.f : exp_of<T>((base - st.m) * inv_t)) * kt : 0.f;
        const float f1 = KEEP && M != kOne ? (none ? 0.f : exp_of<T>(base - st.m)) * k1 : 0.f;
#pragma unroll
        for (int u = 0; u < KP; ++u) {
          // Where the packet is converted anew, 32-bit copies kept from above would not fit.
          if constexpr (!KEEP)
            asm volatile("" : "+r"(p[u].u.x), "+r"(p[u].u.y), "+r"(p[u].u.z), "+r"(p[u].u.w));
          PK o;
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            if constexpr (KEEP) {
              const float2 f = e[u][k];
              float2 g = make_float2(both(f.x, ft, f1), both(f.y, ft, f1));
              if constexpr (M == kTwo)
                g = make_float2(fmaf(e1[u][k].x, f1, g.x), fmaf(e1[u][k].y, f1, g.y));
              o.p[k].set(g);
            } else {
              const float2 x = p[u].p[k].f();
              if constexpr (sizeof(T) == 2 && M != kTwo) {
                const float2 c = make_float2(ct_row, ct_row);
                if constexpr (M == kOne) {
                  // (fp16: the maximum as a pair, beside the other two, spills: 249 against 237 us
                  // at 8192 x 32000; bf16: single 788, as a pair 783 at 8192 x 128256.)
                  float2 d = make_float2(x.x - st.m, x.y - st.m);
                  if (std::is_same<T, __nv_bfloat16>::value)
                    d = __fadd2_rn(x, make_float2(-st.m, -st.m));
                  const float2 t = __ffma2_rn(d, c, make_float2(ot, ot));
                  o.p[k].set(make_float2(ex2f(t.x), ex2f(t.y)));
                } else {
                  const float2 t = __fmul2_rn(__fadd2_rn(x, make_float2(-st.m, -st.m)), c);
                  const float2 b = make_float2(ex2f(t.x), ex2f(t.y));
                  const float2 wt = make_float2(kt, kt), w1 = make_float2(k1, k1);
                  if constexpr (M == kPowers) {
                    float2 f, f1;
                    powers_of_pair(b, f, f1);
                    o.p[k].set(__ffma2_rn(f1, w1, __fmul2_rn(f, wt)));
                  } else {
                    o.p[k].set(__fmul2_rn(b, __ffma2_rn(b, w1, wt)));
                  }
                }
              } else {
                o.p[k].set(make_float2(dense(x.x), dense(x.y)));
              }
            }
          }
          if ((u + 1 < KP && most_full) || tid + u * THREADS < sl.count)
            __stcs(out + u * THREADS, o.u);
        }
        if (xs_at >= 0) dst[xs_at] = Elt<T>::from_f(dense(xs));
      }
    }
    __syncthreads();  // the listed places are written over the dense values
    // The listed elements of this CTA: their part of the loss, and their gradient.  A part whose
    // weight is 0 is left out, even where it is infinite or NaN.
    float l = 0.f;
    auto listed = [&](int j, int c, float x, float pj) {
      const float d = x - st.m;
      const bool label = j == a.list - 1;
      if (sw > 0.f && pj != 0.f) l -= sw * a.temperature * pj * d;
      if (hw > 0.f && label) l -= hw * d;
      if (grad) {
        float g = kt * exp_of<T>(d * inv_t) - (sw > 0.f ? ct * pj : 0.f);
        if constexpr (M != kOne) g = fmaf(k1, exp_of<T>(d), g);
        if (label) g -= c1;
        dst[c] = Elt<T>::from_f(g);
      }
    };
    if (!plain && lists) {
      if (has) listed(tid, id, x_id, p_id);
      for (int j = tid + THREADS; j < a.list; j += THREADS) {
        const int c = a.ids[(int64_t)row * a.list + j];
        if (mine(c)) listed(j, c, picked[j], a.probs[(int64_t)row * a.list + j]);
      }
      total += (double)l;
    }
    if (rank == 0 && tid == THREADS - 1) {
      if (plain) l = fill;
      else {
        l = 0.f;
        if (sw > 0.f) l = sw * a.temperature * a.temperature * (row_entropy + logf(st.z));
        if (hw > 0.f) l += hw * logf(M != kOne ? st.z1 : st.z);
      }
      total += (double)l;
    }
    if (++q == stages) {
      q = 0;
      phase ^= 1;
    }
    xphase ^= xb;
    xb ^= 1;
    src += step * lstride;
    dst += step * gstride;
    if (!same_slice) sl = slice_of(src);
  }
  if (!ok) {  // the loss is poisoned too; what may still be on its way is waited for once more
    total = __longlong_as_double(0x7ff8000000000000ll);
    for (int i = 0; i < 2 * stages; ++i) ptx::mbar_wait(&full[i >> 1], (uint32_t)(i & 1), kPolls);
  }
  if (C > 1) ptx::cluster_sync();  // nobody's shared memory is written after its CTA is gone
  finish_loss(a, total);
}

template <typename T, Mode M, bool KEEP, int THREADS, int KP, int MIN_CTAS>
int launch_rows(const T* lp, int64_t ls, T* gp, int64_t gs, int log_c, int stage_bytes,
                const RowArgs& a, cudaStream_t st) {
  constexpr auto kern = distill_rows<T, M, KEEP, THREADS, KP, MIN_CTAS>;
  const int list_bytes = (a.list + 3) / 4 * 16;
  // As many stages as leave room for MIN_CTAS on an SM (227 KB less 1 KB and the static part).
  int stages = ((227 * 1024) / MIN_CTAS - 2048 - list_bytes) / stage_bytes;
  stages = stages < 1 ? 1 : stages > kMaxStages ? kMaxStages : stages;
  const int smem = stages * stage_bytes + list_bytes;
  allow_shared_memory<kern>(2048);
  const int cluster = 1 << log_c;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // The grid is what the GPU holds at once (clusters of 8 do not fill every SM).
  // The last answer of this thread is kept: it depends on the device and these sizes alone.
  static thread_local int asked_dev = -1, asked_smem, asked_cluster, answer;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (asked_dev != dev || asked_smem != smem || asked_cluster != cluster) {
    if (cudaOccupancyMaxActiveClusters(&answer, kern, &cfg) != cudaSuccess || answer < 1) {
      cudaGetLastError();
      answer = 1;
    }
    asked_dev = dev;
    asked_smem = smem;
    asked_cluster = cluster;
  }
  int most = answer;
  if (most * cluster > num_sms() * kMaxRowCtasPerSm) most = num_sms() * kMaxRowCtasPerSm / cluster;
  const int64_t clusters = a.n_rows < most ? a.n_rows : most;
  cfg.gridDim = dim3((unsigned)((clusters < 1 ? 1 : clusters) * cluster));
  // The kernel may start, and load its first rows, while the teacher kernel ends.  Not so a
  // grid of clusters that fills the GPU: placed among the teacher's last CTAs it finds no room
  // for all its clusters at once, and the rest runs as a second wave (1186 against 717 us at
  // 8192 x 128256 bf16).
  if (cluster == 1 || 2 * clusters <= most) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, lp, ls, gp, gs, stage_bytes, stages, log_c, a);
  if (e != cudaSuccess) return fail(FK_ERR_LAUNCH, "fk_distill(rows): %s", cudaGetErrorString(e));
  return launch_status("fk_distill(rows)");
}

template <typename T, Mode M>
int rows_mode(const T* lp, int64_t ls, T* gp, int64_t gs, const RowArgs& a, cudaStream_t st) {
  // Cluster: as many CTAs as a row needs for slices of at most 32 KB (64 KB where 8 do not
  // suffice), more (down to 8 KB) while the rows are too few for the SMs.  128 threads of 16
  // packets and 4 such CTAs per SM measured best at 8192 x 128256 bf16: 717 us (725 since x - max
  // is formed), against 809 with 256 threads and half the CTAs per row, 942 with 256 threads of 8
  // packets.
  const int64_t packets = (int64_t)a.n_cols * sizeof(T) / 16 + 1;
  int lc = 0;
  while (lc < 3 && packets > (int64_t)2048 << lc) ++lc;
  while (lc < 3 && (a.n_rows << lc) < num_sms() && (packets >> lc) > 512) ++lc;
  const int64_t per = (packets + ((int64_t)1 << lc) - 1) >> lc;
  const int bytes = (int)(per < 1 ? 16 : per * 16);
  constexpr bool keep = sizeof(T) == 4 && (M == kOne || M == kSquare);
  if (per <= 128) return launch_rows<T, M, true, 128, 1, 8>(lp, ls, gp, gs, lc, bytes, a, st);
  if (per <= 512) return launch_rows<T, M, keep, 128, 4, 8>(lp, ls, gp, gs, lc, bytes, a, st);
  if (per <= 2048) return launch_rows<T, M, keep, 128, 16, 4>(lp, ls, gp, gs, lc, bytes, a, st);
  return launch_rows<T, M, keep, 256, 16, 2>(lp, ls, gp, gs, lc, bytes, a, st);
}

template <typename T>
int rows_t(const void* logits, int64_t ls, void* grad, int64_t gs, const RowArgs& a,
           cudaStream_t st) {
  const T* lp = static_cast<const T*>(logits);
  T* gp = static_cast<T*>(grad);
  const int64_t apart = reinterpret_cast<intptr_t>(lp) - reinterpret_cast<intptr_t>(gp);
  const bool same_offset = !gp || (apart % 16 == 0 && (ls - gs) * (int64_t)sizeof(T) % 16 == 0);
  const int64_t packets = (int64_t)a.n_cols * sizeof(T) / 16 + 1;
  if (same_offset && packets <= 8 * 4096) {
    RowArgs b = a;
    if (a.hard_weight == 1.f) b.temperature = b.inv_t = 1.f;  // the soft part has no weight
    if (b.temperature == 1.f || a.hard_weight == 0.f)
      return rows_mode<T, kOne>(lp, ls, gp, gs, b, st);
    if (b.temperature == 2.f) return rows_mode<T, kSquare>(lp, ls, gp, gs, b, st);
    b.q2 = b.temperature == 1.5f;
    b.p4 = b.temperature == 4.f;
    b.inv_p = b.p4 ? 0.25f : 1.0f / 3.0f;
    if (b.q2 || b.p4 || b.temperature == 3.f) return rows_mode<T, kPowers>(lp, ls, gp, gs, b, st);
    return rows_mode<T, kTwo>(lp, ls, gp, gs, b, st);
  }
  const int64_t most = (int64_t)num_sms() * 8;
  const int grid = (int)(a.n_rows < most ? a.n_rows : most);
  distill_rows_generic<T><<<grid < 1 ? 1 : grid, kGenericThreads, 0, st>>>(lp, ls, gp, gs, a);
  return launch_status("fk_distill(rows)");
}

template <typename T>
int teacher_t(const int64_t* idx, const void* top, int k, const int64_t* targets,
              int64_t ignore_index, int64_t n_rows, int64_t n_cols, float inv_t,
              const Workspace& ws, int* ctas, cudaStream_t st) {
  int log_table = 5;
  while ((1 << log_table) < 2 * k) ++log_table;
  // Many short rows: 8 lanes a row, so that the reductions of 4 rows are one instruction.  Few
  // or long ones: a warp a row.  8 lanes against a warp, us: 8192 rows of 16 5.7 / 7.9, 8192 of 64
  // 11.3 / 10.4, 32768 of 64 24.9 / 33.5; 2048 of 16 5.3 / 5.0, 2048 of 64 10.0 / 6.1, 8192 of 100
  // 15.4 / 15.2; at the edge itself, 4096 of 64, 10.5 / 7.4.
  const bool narrow = n_rows >= 4096 && k <= 64;
  const int rows = kTeacherWarps * (narrow ? 4 : 1);
  const int smem = rows * row_ints(k, log_table) * 4;
  const int64_t want = (n_rows + rows - 1) / rows;
  *ctas = (int)(want < 1 ? 1 : want > kTeacherCtas ? kTeacherCtas : want);
  auto launch = [&](auto kern) {
    kern<<<*ctas, kTeacherWarps * 32, smem, st>>>(idx, static_cast<const T*>(top), k, log_table,
                                                  targets, ignore_index, (int)n_rows, n_cols,
                                                  inv_t, ws);
  };
  allow_shared_memory<distill_teacher<T, 32>>(1024);  // 8 lanes a row stay below 48 KB
  if (narrow) launch(distill_teacher<T, 8>);
  else launch(distill_teacher<T, 32>);
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
  FK_CHECK_ARG(n_rows < ((int64_t)1 << 31) - 65536, "fk_distill: n_rows too large");
  if (k > fk::kMaxSlots)
    return fk::fail(FK_ERR_UNSUPPORTED, "fk_distill: k=%d exceeds %d", k, fk::kMaxSlots);
  FK_CHECK_ARG(fk::valid_dtype(dtype) && fk::valid_dtype(teacher_dtype), "fk_distill: bad dtype");
  FK_CHECK_ARG(row_stride >= n_cols && (!grad || grad_row_stride >= n_cols),
               "fk_distill: stride < n_cols");
  FK_CHECK_ARG(temperature > 0.f && temperature < INFINITY, "fk_distill: temperature must be > 0");
  FK_CHECK_ARG(hard_weight >= 0.f && hard_weight <= 1.f, "fk_distill: hard_weight outside [0, 1]");
  FK_CHECK_ARG(loss_scale > 0.f && loss_scale < INFINITY, "fk_distill: loss_scale must be > 0");
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
  a.sums = ws.sums;
  a.ticket = ws.ticket;
  a.loss = loss;
  a.err = err_flag;
  a.list = k + 1;
  a.n_cols = (int)n_cols;
  a.n_rows = n_rows;
  a.temperature = temperature;
  a.inv_t = 1.0f / temperature;
  a.inv_p = 1.f;
  a.q2 = a.p4 = false;
  a.hard_weight = targets ? hard_weight : 0.f;
  a.loss_scale = loss_scale;
  FK_DISPATCH_DTYPE(dtype, s = fk::rows_t<scalar_t>(logits, row_stride, grad, grad_row_stride, a,
                                                    st));
  return s;
}
