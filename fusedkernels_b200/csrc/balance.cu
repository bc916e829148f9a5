// Router balance loss, z-loss and per-expert counts, with the gradient.
//
//   c_e = #slots of counted tokens that name expert e,  f_e = c_e / max(1, sum c),
//   p_t = softmax(logits_t),  S_t = sum_e f_e p_te,  n = max(1, #counted tokens)
//   loss = E/n * sum_t S_t + z/n * sum_t lse_t^2
//   dloss/dlogits_te = p_te * (E/n * (f_e - S_t) + 2 z/n * lse_t)
//
// As the p_te of a token add up to 1, f may be centred: with g_e = f_e - 1/E (formed from the
// counts, where it is exact) S_t = 1/E + sum_e g_e p_te and f_e - S_t = g_e - sum_j g_j p_tj.  That
// keeps the gradient's bits where the load is nearly even and f_e and S_t nearly cancel.
//
// f depends on the slots alone, so a first small kernel counts them and the second reads
// every logit once and writes its gradient at once: the logits are not read again in a
// backward pass.  The counts are integers and the loss is summed in a fixed order, so
// results do not depend on the order in which CTAs run.
#include "common.cuh"
#include "exp.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace fk {
namespace {

constexpr int kMaxExperts = 256;
constexpr int kCountClusters = 16;  // partial histograms that every CTA of the second kernel adds up
constexpr int kCountCluster = 8;    // CTAs that make one partial histogram
constexpr int kCountThreads = 512;
constexpr int kCountStride = kMaxExperts + 4;  // E counts, then the counted tokens, then bad slots
constexpr int kMainThreads = 256;
constexpr int kMainWarps = kMainThreads / 32;
constexpr int kMainCtasPerSm = 8;

struct Workspace {
  int* part;      // [kCountClusters][kCountStride]
  double2* sums;  // [main grid] (sum S, sum lse^2)
  unsigned* ticket;
};

inline size_t ws_bytes() {
  return (size_t)kCountClusters * kCountStride * sizeof(int) +
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

// Slots are counted in shared memory, the CTAs of a cluster add their counts up over its shared
// memories, and one partial histogram per cluster leaves (the second kernel's CTAs each read all
// of them: with one per CTA that took longer than their rows at 20011 tokens).  Two slots a
// load where idx allows it, and a thread has eight loads in flight: one after the other they
// took 13.7 of 54 us at 131072 tokens of 8 slots.
__global__ void __cluster_dims__(kCountCluster, 1, 1) __launch_bounds__(kCountThreads)
balance_count(
    const int64_t* __restrict__ idx, const uint8_t* __restrict__ mask, unsigned n_rows, unsigned k,
    int n_experts, int pairs, int* __restrict__ part, unsigned* __restrict__ ticket) {
  __shared__ int hist[kCountStride];
  ptx::let_next_kernel_start();
  for (int i = threadIdx.x; i < kCountStride; i += kCountThreads) hist[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  __syncthreads();
  const unsigned me = blockIdx.x * kCountThreads + threadIdx.x, step = gridDim.x * kCountThreads;
  const unsigned slots = n_rows * k;
  int bad = 0;
  auto count = [&](unsigned slot, int64_t e) {
    if (mask && !mask[slot / k]) return;
    if ((uint64_t)e < (uint64_t)n_experts) atomicAdd(&hist[(int)e], 1);
    else bad += e >= 0;
  };
  const unsigned paired = pairs ? slots / 2 : 0;
  constexpr int kBatch = 8;
  for (unsigned i0 = me; i0 < paired; i0 += kBatch * step) {
    longlong2 e[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      e[b] = make_longlong2(-1, -1);
      if (i0 + b * step < paired) e[b] = __ldg(reinterpret_cast<const longlong2*>(idx) + i0 + b * step);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const unsigned i = i0 + b * step;
      if (i < paired) {
        count(2 * i, e[b].x);
        count(2 * i + 1, e[b].y);
      }
    }
  }
  for (unsigned i = 2 * paired + me; i < slots; i += step) count(i, __ldg(idx + i));
  int tokens = 0;
  if (mask)
    for (unsigned t = me; t < n_rows; t += step) tokens += mask[t] != 0;
  else if (me == 0)
    tokens = (int)n_rows;
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  bad = __reduce_add_sync(0xffffffffu, bad);
  if ((threadIdx.x & 31) == 0) {
    if (tokens) atomicAdd(&hist[n_experts], tokens);
    if (bad) atomicAdd(&hist[n_experts + 1], bad);
  }
  ptx::cluster_sync();
  // CTA r of the cluster adds up the entries r, r + 8, ...
  const int rank = (int)ptx::cluster_ctarank();
  for (int i = rank + kCountCluster * threadIdx.x; i < n_experts + 2;
       i += kCountCluster * kCountThreads) {
    int sum = 0;
#pragma unroll
    for (int c = 0; c < kCountCluster; ++c)
      sum += ptx::ld_dsmem_s32(ptx::peer_smem(&hist[i], (uint32_t)c));
    part[(blockIdx.x / kCountCluster) * kCountStride + i] = sum;
  }
  ptx::cluster_sync();  // no CTA's shared memory goes before it has been read
}

// A lane's share of a token's logits (-inf past the row's end).  PACKED: L lanes a token, lane l
// has its 16-byte packets l, l + L, ...; else a warp a token, lane l the elements l, l + 32, ...
template <typename T, bool PACKED, int L, int PP>
struct Share {
  static constexpr int VN = PACKED ? 16 / (int)sizeof(T) : 1;
  static constexpr int N = PP * VN;
  Vec16<T> p[PACKED ? PP : 1];
  T e[PACKED ? 1 : PP];
  __device__ __forceinline__ Share() {}
  __device__ __forceinline__ void load(const T* row, int l, int n, bool on) {
#pragma unroll
    for (int u = 0; u < PP; ++u) {
      const int c = (l + u * L) * VN;
      if constexpr (PACKED) {
        constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u
                               : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        p[u].u = make_uint4(w, w, w, w);
        if (on && c < n) p[u] = ld_stream(row + c);
      } else {
        e[u] = Elt<T>::from_f(-INFINITY);
        if (on && c < n) e[u] = row[c];
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (PACKED) return Elt<T>::to_f(p[i / VN].e[i % VN]);
    else return Elt<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void put(int i, float v) {
    if constexpr (PACKED) p[i / VN].e[i % VN] = Elt<T>::from_f(v);
    else e[i] = Elt<T>::from_f(v);
  }
  __device__ __forceinline__ void store(T* row, int l, int n) const {
#pragma unroll
    for (int u = 0; u < PP; ++u) {
      const int c = (l + u * L) * VN;
      if (c < n) {
        if constexpr (PACKED) st_stream(row + c, p[u]);
        else row[c] = e[u];
      }
    }
  }
  // The entries of table f (kMaxExperts of them) for this lane's elements.
  static __device__ __forceinline__ void table(const float* f, int l, float (&out)[N]) {
#pragma unroll
    for (int u = 0; u < PP; ++u) {
      const int c = (l + u * L) * VN & (kMaxExperts - 1);
      if constexpr (PACKED) {
#pragma unroll
        for (int k = 0; k < VN; k += 4) {
          const float4 v = *reinterpret_cast<const float4*>(f + c + k);
          out[u * VN + k] = v.x;
          out[u * VN + k + 1] = v.y;
          out[u * VN + k + 2] = v.z;
          out[u * VN + k + 3] = v.w;
        }
      } else {
        out[u] = f[c];
      }
    }
  }
};

// How the rows of logits are read.
//   kPacked  rows of whole 16-byte packets: 8 or 16 lanes a token, packets to registers;
//   kTiled   contiguous rows of any width: 16 / sizeof(T) rows are whole packets together, a
//            warp brings them through its part of shared memory, 8 lanes a token;
//   kSingle  other strides: a warp a token, single elements.
enum Layout { kPacked, kTiled, kSingle };

// What the rows need to know of the counts.
struct Frame {
  float f[kMaxExperts];  // share of the slots less 1/E (NaN after an index out of range)
  int tot[kCountStride];
  int slots;
  double2 red[kMainWarps];
  bool last;
};

// Adds up the partial histograms (all threads; after the counting kernel is done).
__device__ __forceinline__ void read_counts(Frame& fr, const int* part, int n_parts,
                                            int n_experts, int64_t* counts) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kCountStride; i += kMainThreads) fr.tot[i] = 0;
  if (tid == 0) fr.slots = 0;
  __syncthreads();
  constexpr int kQuads = kCountStride / 4;
  const int quads = (n_experts + 2 + 3) / 4;
#pragma unroll 8
  for (int i = tid; i < n_parts * quads; i += kMainThreads) {
    const int g = i / quads, c = i % quads;
    const int4 v = __ldcg(reinterpret_cast<const int4*>(part) + g * kQuads + c);
    if (v.x) atomicAdd(&fr.tot[4 * c], v.x);
    if (v.y) atomicAdd(&fr.tot[4 * c + 1], v.y);
    if (v.z) atomicAdd(&fr.tot[4 * c + 2], v.z);
    if (v.w) atomicAdd(&fr.tot[4 * c + 3], v.w);
  }
  __syncthreads();
  const int mine = __reduce_add_sync(0xffffffffu, tid < n_experts ? fr.tot[tid] : 0);
  if ((tid & 31) == 0) atomicAdd(&fr.slots, mine);
  __syncthreads();
  const int c = tid < n_experts ? fr.tot[tid] : 0;
  const double slots = (double)(fr.slots < 1 ? 1 : fr.slots);  // none used: c - slots is 0 too
  fr.f[tid] = fr.tot[n_experts + 1]
                  ? __int_as_float(0x7fc00000)
                  : (float)(((double)c * n_experts - (double)fr.slots) / (slots * n_experts));
  if (blockIdx.x == 0 && tid < n_experts) counts[tid] = c;
  __syncthreads();
}
static_assert(kMainThreads == kMaxExperts, "a thread per expert in read_counts");

// Softmax of one token over L lanes with N logits each (-inf past the end): v becomes
// exp(v - max); returns 1 / sum (0 where there is none), the token's sum of f p and its
// logsumexp.
template <int L, int N>
__device__ __forceinline__ float token(float (&v)[N], const float (&f)[N], float& s, float& lse) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);  // a NaN comes back in the sum
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float top = m == -INFINITY ? 0.f : m;
  float z = 0.f;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = exp2_of(v[i] - top);
    z += v[i];
    s = fmaf(v[i], f[i], s);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  // A row of -inf alone has no probabilities: it adds nothing and gets no gradient.
  const float inv = z == 0.f ? 0.f : 1.0f / z;
  lse = z == 0.f ? 0.f : top + logf(z);
  s *= inv;
  return inv;
}

struct Args {
  const void* logits;
  int64_t stride;
  const int64_t* idx;
  const uint8_t* mask;
  int n_rows, n_experts, k;
  float z_coef, loss_scale;
  void* grad;
  int64_t* counts;
  float* loss;
};

// Rows are read ahead: the next ones are on their way while these are worked on, and the first
// ones while the counting kernel ends.  At 131072 x 128 fp32 25 us by itself, 32 from its start
// under the count (its floor is 21: the copy rate); 62% of the issue slots, 26 instructions a
// logit and warp, so it is bound by both.  Count and rows together there: 37 us with three CTAs an
// SM (24 bytes spilled), 37 with two (none), 43 with four.
template <typename T, Layout LAYOUT, int L, int PP>
constexpr int ctas_per_sm() {  // by the registers that a lane's logits take
  const int values = LAYOUT == kPacked ? PP * 16 / (int)sizeof(T) : LAYOUT == kTiled ? 4 * PP : PP;
  return values <= 8 ? 4 : values <= 16 ? 3 : 2;
}
template <typename T, Layout LAYOUT, int L, int PP>
__global__ void __launch_bounds__(kMainThreads, ctas_per_sm<T, LAYOUT, L, PP>()) balance_main(Args a, const int* part,
                                                             int n_parts, double2* sums,
                                                             unsigned* ticket) {
  extern __shared__ __align__(16) unsigned char tiles[];
  __shared__ __align__(16) Frame fr;
  const T* logits = static_cast<const T*>(a.logits);
  T* grad = static_cast<T*>(a.grad);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L, n_experts = a.n_experts;
  const int gw = (int)blockIdx.x * kMainWarps + warp, warps = (int)gridDim.x * kMainWarps;
  double sum_s = 0.0, sum_z = 0.0;
  float ce = 0.f, cz = 0.f, even = 0.f;
  auto start = [&] {
    ptx::wait_for_previous_kernel();
    read_counts(fr, part, n_parts, n_experts, a.counts);
    const float n = (float)(fr.tot[n_experts] < 1 ? 1 : fr.tot[n_experts]);
    ce = (float)n_experts * a.loss_scale / n;
    cz = 2.f * a.z_coef * a.loss_scale / n;
    even = fr.slots < 1 ? 0.f : 1.0f / (float)n_experts;
  };
  auto add = [&](bool on, float inv, float s, float lse) {
    if (l == 0 && on && inv != 0.f) {  // (true for NaN)
      sum_s += (double)even + (double)s;
      sum_z += (double)lse * (double)lse;
    }
  };
  if constexpr (LAYOUT == kTiled) {
    // Tile: kRows rows, a multiple of 16 bytes.  PP packets a lane hold it.
    constexpr int kRows = 16 / (int)sizeof(T), kPer = 32 * PP / L;
    T* tile = reinterpret_cast<T*>(tiles + (size_t)warp * n_experts * 16);
    uint4 next[PP];
    auto load = [&](int t) {
      if ((t + 1) * kRows > a.n_rows) return;
      const uint4* src = reinterpret_cast<const uint4*>(logits + (int64_t)t * kRows * n_experts);
#pragma unroll
      for (int u = 0; u < PP; ++u)
        if (lane + 32 * u < n_experts) next[u] = __ldcs(src + lane + 32 * u);
    };
    load(gw);
    start();
    for (int t = gw; t * kRows < a.n_rows; t += warps) {
      if ((t + 1) * kRows <= a.n_rows) {
#pragma unroll
        for (int u = 0; u < PP; ++u)
          if (lane + 32 * u < n_experts) reinterpret_cast<uint4*>(tile)[lane + 32 * u] = next[u];
      } else {  // the last rows, fewer than a tile: single elements
        const T* src = logits + (int64_t)t * kRows * n_experts;
        for (int i = lane; i < (a.n_rows - t * kRows) * n_experts; i += 32) tile[i] = src[i];
      }
      __syncwarp();
      load(t + warps);
#pragma unroll 1
      for (int g = lane / L; g < kRows; g += 32 / L) {
        const int row = t * kRows + g;
        const bool on = row < a.n_rows && (!a.mask || a.mask[row]);
        T* at = tile + g * n_experts + l;
        float v[kPer], f[kPer], s, lse;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          v[i] = on && l + i * L < n_experts ? Elt<T>::to_f(at[i * L]) : -INFINITY;
          f[i] = fr.f[l + i * L];
        }
        const float inv = token<L, kPer>(v, f, s, lse);
        add(on, inv, s, lse);
        const float c0 = on ? inv * fmaf(cz, lse, -ce * s) : 0.f, c1 = on ? inv * ce : 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (l + i * L < n_experts) at[i * L] = Elt<T>::from_f(v[i] * fmaf(c1, f[i], c0));
      }
      __syncwarp();
      if (grad) {
        T* dst = grad + (int64_t)t * kRows * n_experts;
        const int rows = a.n_rows - t * kRows;
        const int left = (rows < kRows ? rows : kRows) * n_experts;  // elements of the tile
        for (int u = lane; u < n_experts; u += 32) {
          if ((u + 1) * kRows <= left)
            __stcs(reinterpret_cast<uint4*>(dst) + u, reinterpret_cast<const uint4*>(tile)[u]);
          else
            for (int k = u * kRows; k < left; ++k) dst[k] = tile[k];
        }
      }
      __syncwarp();
    }
  } else {
    using S = Share<T, LAYOUT == kPacked, L, PP>;
    constexpr int kTokens = 32 / L;  // of a warp at a time
    S cur, next;
    bool next_on = false;
    auto load = [&](int row) {
      next_on = row < a.n_rows && (!a.mask || a.mask[row]);
      next.load(logits + row * a.stride, l, n_experts, next_on);
    };
    load(gw * kTokens + lane / L);
    start();
    for (int base = gw * kTokens; base < a.n_rows; base += warps * kTokens) {
      const int row = base + lane / L;
      const bool on = next_on;
      cur = next;
      load(row + warps * kTokens);
      float v[S::N], f[S::N], s, lse;
#pragma unroll
      for (int i = 0; i < S::N; ++i) v[i] = cur.get(i);
      S::table(fr.f, l, f);
      const float inv = token<L, S::N>(v, f, s, lse);
      add(on, inv, s, lse);
      if (grad && row < a.n_rows) {
        const float c0 = on ? inv * fmaf(cz, lse, -ce * s) : 0.f, c1 = on ? inv * ce : 0.f;
#pragma unroll
        for (int i = 0; i < S::N; ++i) cur.put(i, v[i] * fmaf(c1, f[i], c0));
        cur.store(grad + (int64_t)row * n_experts, l, n_experts);
      }
    }
  }
  auto block_total = [&](double2 x) {  // fixed order; valid in thread 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
      x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
    }
    __syncthreads();
    if (lane == 0) fr.red[warp] = x;
    __syncthreads();
    x = fr.red[0];
    for (int i = 1; i < kMainWarps; ++i) {
      x.x += fr.red[i].x;
      x.y += fr.red[i].y;
    }
    return x;
  };
  double2 x = block_total(make_double2(sum_s, sum_z));
  if (threadIdx.x == 0) {
    sums[blockIdx.x] = x;
    __threadfence();
    fr.last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!fr.last) return;
  __threadfence();
  x = make_double2(0.0, 0.0);
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kMainThreads) {
    x.x += __ldcg(&sums[i].x);
    x.y += __ldcg(&sums[i].y);
  }
  x = block_total(x);
  if (threadIdx.x == 0) {
    const double n = (double)(fr.tot[n_experts] < 1 ? 1 : fr.tot[n_experts]);
    *a.loss = fr.tot[n_experts + 1]
                  ? __int_as_float(0x7fc00000)
                  : (float)(((double)n_experts * x.x + (double)a.z_coef * x.y) / n);
  }
}

template <typename T, Layout LAYOUT, int L, int PP>
int main_t(const Args& a, const Workspace& ws, int n_parts, cudaStream_t st) {
  constexpr auto kern = balance_main<T, LAYOUT, L, PP>;
  const int smem = LAYOUT == kTiled ? kMainWarps * a.n_experts * 16 : 0;  // at most 32 KB
  static thread_local int asked_dev = -1, asked_smem, per_sm;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (asked_dev != dev || asked_smem != smem) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kMainThreads,
                                                      (size_t)smem) != cudaSuccess ||
        per_sm < 1) {
      cudaGetLastError();
      per_sm = 1;
    }
    if (per_sm > kMainCtasPerSm) per_sm = kMainCtasPerSm;
    asked_dev = dev;
    asked_smem = smem;
  }
  const int tokens = kMainWarps * (LAYOUT == kTiled ? 16 / (int)sizeof(T) : 32 / L);
  const int want = (a.n_rows + tokens - 1) / tokens, most = num_sms() * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(want < 1 ? 1 : want < most ? want : most));
  cfg.blockDim = dim3(kMainThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, kern, a, (const int*)ws.part, n_parts, ws.sums, ws.ticket);
  if (e != cudaSuccess) return fail(FK_ERR_LAUNCH, "fk_moe_balance: %s", cudaGetErrorString(e));
  return launch_status("fk_moe_balance");
}

template <typename T>
int fwd_t(const Args& a, void* workspace, cudaStream_t st) {
  const Workspace ws = ws_split(workspace);
  constexpr int64_t per = 4 * kCountThreads * kCountCluster;  // slots a cluster is worth
  const int64_t g = ((int64_t)a.n_rows * a.k + per - 1) / per;
  const int n_parts = (int)(g < 1 ? 1 : g > kCountClusters ? kCountClusters : g);
  balance_count<<<n_parts * kCountCluster, kCountThreads, 0, st>>>(a.idx, a.mask, (unsigned)a.n_rows,
                                                      (unsigned)a.k, a.n_experts,
                                                      aligned16(a.idx), ws.part, ws.ticket);
  int s = launch_status("fk_moe_balance(count)");
  if (s != FK_OK) return s;
  constexpr int VN = 16 / (int)sizeof(T);
  const bool aligned = aligned16(a.logits) && aligned16(a.grad);
  const int e = a.n_experts;
  if (aligned && e % VN == 0 && a.stride % VN == 0) {
    if (e <= 8 * VN) return main_t<T, kPacked, 8, 1>(a, ws, n_parts, st);
    if (e <= 16 * VN) return main_t<T, kPacked, 8, 2>(a, ws, n_parts, st);
    if (e <= 32 * VN) return main_t<T, kPacked, 8, 4>(a, ws, n_parts, st);
    return main_t<T, kPacked, 16, 4>(a, ws, n_parts, st);
  }
  if (aligned && a.stride == e) {
    if (e <= 64) return main_t<T, kTiled, 8, 2>(a, ws, n_parts, st);
    if (e <= 128) return main_t<T, kTiled, 8, 4>(a, ws, n_parts, st);
    if (e <= 192) return main_t<T, kTiled, 8, 6>(a, ws, n_parts, st);
    return main_t<T, kTiled, 8, 8>(a, ws, n_parts, st);
  }
  if (e <= 64) return main_t<T, kSingle, 32, 2>(a, ws, n_parts, st);
  return main_t<T, kSingle, 32, 8>(a, ws, n_parts, st);
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
  FK_CHECK_ARG(n_rows * (int64_t)(k < 1 ? 1 : k) < ((int64_t)1 << 31) - (1 << 22),
               "fk_moe_balance: nearly 2^31 slots or more");
  FK_CHECK_ARG(row_stride >= n_experts, "fk_moe_balance: stride < n_experts");
  FK_CHECK_ARG(fk::valid_dtype(dtype), "fk_moe_balance: bad dtype code %d", dtype);
  FK_CHECK_ARG(loss_scale > 0.f && loss_scale < INFINITY, "fk_moe_balance: loss_scale must be > 0");
  FK_CHECK_ARG(counts && loss, "fk_moe_balance: null pointer");
  FK_CHECK_ARG(n_rows == 0 || (logits && (idx || k == 0)), "fk_moe_balance: null pointer");
  if (workspace == nullptr || workspace_bytes < fk::ws_bytes() || !fk::aligned16(workspace))
    return fk::fail(FK_ERR_WORKSPACE, "fk_moe_balance: need %zu aligned workspace bytes, got %zu",
                    fk::ws_bytes(), workspace_bytes);
  const fk::Args a{logits, row_stride, idx,    token_mask, (int)n_rows, n_experts,
                   k,      z_coef,     loss_scale, grad,   counts,      loss};
  FK_DISPATCH_DTYPE(dtype, return fk::fwd_t<scalar_t>(a, workspace, fk::as_stream(stream)));
  return FK_OK;
}
