// Residual addition + RMSNorm: forward, backward, and a forward with an 8-bit output.
//
//   h = round_R(x + r),  s = rsqrt(mean(h^2) + eps),  y = round_T(h * s * w)
//   given dy, dh:  g = dh + s*w*dy - h * s^3 * mean(w*dy*h),  dx = round_T(g),
//   dr = round_R(g),  dw = sum_rows dy*h*s
//   8 bits: per group of columns  scale = max(max|h*s*w| / 448, 2^-126),
//   q = e4m3(h*s*w / scale) with the fp32 product h*s*w, not its rounding to T.
//
// The norm is taken of the rounded sum h, the tensor that is stored and that the backward
// reads, so forward and backward see the same row.  T is the type of x and y, R the type
// of the residual stream (T or fp32); every statistic is fp32.
#include "common.cuh"
#include "ptx.cuh"

#include <cuda_fp8.h>

namespace fk {
namespace {

constexpr uint32_t kPolls = 1u << 21;  // of a wait, before it gives up
constexpr int kMaxGridPerSm = 8;  // CTAs of a backward grid, and partial rows of dw, per SM
constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: a row of zeros keeps a usable scale

__device__ __forceinline__ float load_wd(const void* w, int wd, int64_t c) {
  if (wd == FK_F32) return static_cast<const float*>(w)[c];
  if (wd == FK_F16) return Elt<__half>::to_f(static_cast<const __half*>(w)[c]);
  return Elt<__nv_bfloat16>::to_f(static_cast<const __nv_bfloat16*>(w)[c]);
}

__device__ __forceinline__ float block_sum(float v, float* red /*[32]*/) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < nwarps; ++i) s += red[i];  // fixed order: deterministic
  return s;
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float m = red[0];
  for (int i = 1; i < nwarps; ++i) m = fmaxf(m, red[i]);
  return m;
}

// The 8-bit form divides twice: scale = m / 448 for a group's largest magnitude m, and y / scale.
// Products with a reciprocal are off by up to 3 steps, and beside an e4m3 tie that moves a value
// to the other neighbour, a step of up to 1/8 of it.  The residual r = q b - a of such a quotient
// q of a / b is an FMA without error (or next to none), and puts it right (Markstein 1990):
// q - r / b is off by 2^-20 steps before its one rounding, and keeps the sign of a zero.  (A call at
// 16384 x 4096 bf16, per 128: 79 us with the bare products, 80 so, 97 with divisions.)
__device__ __forceinline__ float divide(float a, float b, float inv_b) {
  const float q = a * inv_b;
  return fmaf(-fmaf(q, b, -a), inv_b, q);
}

// (Below kMinScale the residual may leave the normal range, and the quotient is not used.)
__device__ __forceinline__ float scale_of(float m) {
  return m < INFINITY ? fmaxf(divide(m, kE4m3Max, 1.0f / kE4m3Max), kMinScale) : m;
}

// y / scale for the values of a group: of both times a power of two, exactly, where scale is so
// small that residuals would leave the normal range.  (Beside an infinite value q is 0, as by a
// division.)
struct Quotient {
  float by, b, inv;
  __device__ __forceinline__ explicit Quotient(float scale)
      : by(scale < 0x1p-64f ? 0x1p64f : 1.0f), b(scale < INFINITY ? scale * by : 0.f) {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(b));
    if (b == 0.f) inv = 0.f;
  }
  __device__ __forceinline__ float operator()(float y) const { return divide(y * by, b, inv); }
};

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// ------------------------------------------------------------------ 16-byte chunks ------
// A chunk is 16 bytes of x (VN elements) and the same elements of the residual: one 16-byte
// load, or two where the residual is fp32 beside 16-bit x.  A chunk of one element (VN = 1)
// serves rows of any width and alignment.
template <typename R, int VN>
struct Chunk {
  static constexpr int N16 = VN * (int)sizeof(R) / 16;
  union {
    uint4 u[N16 > 0 ? N16 : 1];
    R e[VN];
  };
  __device__ __forceinline__ Chunk() {}
  __device__ __forceinline__ void load(const R* p) {
    if constexpr (VN == 1) e[0] = *p;
#pragma unroll
    for (int i = 0; i < N16; ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(R* p) const {
    if constexpr (VN == 1) *p = e[0];
#pragma unroll
    for (int i = 0; i < N16; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, u[i]);
  }
};

// VN weights from column c on (a multiple of VN), in fp32; they stay in L1 from row to row.
template <int VN>
__device__ __forceinline__ void load_weights(const void* w, int wd, int c, float (&out)[VN]) {
  if constexpr (VN == 1) {
    out[0] = load_wd(w, wd, c);
    return;
  }
  if (wd == FK_F32) {
#pragma unroll
    for (int i = 0; i < VN; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c + i));
      out[i] = f.x;
      out[i + 1] = f.y;
      out[i + 2] = f.z;
      out[i + 3] = f.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VN; i += 4) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + c + i));
    const uint32_t h[2] = {u.x, u.y};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned short b = (unsigned short)(h[k >> 1] >> (16 * (k & 1)));
      out[i + k] = wd == FK_F16 ? __half2float(__ushort_as_half(b))
                                : __bfloat162float(__ushort_as_bfloat16(b));
    }
  }
}

// Sum (or maximum) over the TPR threads that share a row; all of them get it.  Groups of more
// than a warp are whole CTAs.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
    const float b = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, b) : v + b;
  }
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[lane % (TPR / 32)];  // fixed order: deterministic
#pragma unroll
    for (int o = TPR / 64; o > 0; o >>= 1) {
      const float b = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? fmaxf(v, b) : v + b;
    }
  }
  return v;
}

constexpr int fwd_groups(int tpr) { return tpr <= 32 ? 256 / tpr : 1; }

// Forward, and with QUANT the 8-bit form (BLOCK: a scale per 128 columns, else per row).  TPR
// threads take a row, thread t its chunks t, t + TPR, ...: every load of the row is in flight
// before the first is used, the sum h stays in registers, and as the rows are independent the
// SM hides one CTA's reduction under the others' loads.  Bound by HBM: 84 us forward at
// 16384 x 4096 bf16 (6.4 TB/s); in 8 bits 79 us per 128 columns and 82 per row (5.9 and 5.7 TB/s:
// the quotients take the kernel to 85% of the issue slots).  As single elements 16 us at
// 5003 x 1111 bf16 with an fp32 residual (4.2 TB/s; the element loops below 29, whole-line tiles
// through shared memory 32: too few rows in flight), in 8 bits 27 (one byte a store).
template <typename T, typename R, int VN, int TPR, int CPT, bool QUANT, bool BLOCK>
__global__ void __launch_bounds__(TPR <= 32 ? 256 : TPR) add_rmsnorm_rows(
    const T* __restrict__ x, int64_t xs, const R* __restrict__ r, int64_t rs,
    const void* __restrict__ w, int wd, T* __restrict__ y, uint8_t* __restrict__ q,
    float* __restrict__ scales, R* __restrict__ h, float* __restrict__ rstd, int64_t rows,
    int cols, float eps) {
  __shared__ float red[2][32];
  __shared__ float group_max[VN == 1 && BLOCK ? CPT : 1][32];  // by warps
  const int t = threadIdx.x % TPR;
  const int64_t row0 = (int64_t)blockIdx.x * fwd_groups(TPR) + threadIdx.x / TPR;
  const bool there = TPR > 32 || row0 < rows;
  const int64_t row = there ? row0 : rows - 1;  // idle groups go along on the last row
  const int chunks = cols / VN;
  Chunk<T, VN> xv[CPT];
  Chunk<R, VN> hv[CPT];
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = t + u * TPR;
    if (c < chunks) {
      xv[u].load(x + row * xs + c * VN);
      if (r) hv[u].load(r + row * rs + c * VN);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = t + u * TPR;
    if (c < chunks) {
#pragma unroll
      for (int k = 0; k < VN; ++k) {
        float f = Elt<T>::to_f(xv[u].e[k]);
        if (r) {
          hv[u].e[k] = Elt<R>::from_f(f + Elt<R>::to_f(hv[u].e[k]));
          f = Elt<R>::to_f(hv[u].e[k]);
        }
        ss = fmaf(f, f, ss);
      }
      if (r && there) hv[u].store(h + row * cols + c * VN);
    }
  }
  const float s = rsqrtf(row_reduce<TPR, false>(ss, red[0]) / (float)cols + eps);
  if (!QUANT && t == 0 && rstd && there) rstd[row] = s;
  if constexpr (!QUANT) {
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = t + u * TPR;
      if (c < chunks) {
        float wv[VN];
        load_weights<VN>(w, wd, c * VN, wv);
#pragma unroll
        for (int k = 0; k < VN; ++k)
          xv[u].e[k] = Elt<T>::from_f(Elt<R>::to_f(hv[u].e[k]) * s * wv[k]);
        if (there) xv[u].store(y + row * cols + c * VN);
      }
    }
  } else {
    // y of chunk u, and its largest magnitude (0 past the end of the row).
    auto values = [&](int u, float (&y)[VN]) {
      const int c = t + u * TPR;
      float m = 0.f;
      if (c < chunks) {
        load_weights<VN>(w, wd, c * VN, y);
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          y[k] *= (r ? Elt<R>::to_f(hv[u].e[k]) : Elt<T>::to_f(xv[u].e[k])) * s;
          m = fmaxf(m, fabsf(y[k]));
        }
      }
      return m;
    };
    auto put = [&](int u, const float (&y)[VN], const Quotient& quotient) {
      const int c = t + u * TPR;
      if (c >= chunks || !there) return;
      uint8_t* at = q + row * cols + c * VN;
      if constexpr (VN == 1) {
        *at = to_e4m3(quotient(y[0]));
        return;
      }
      uint32_t o[VN > 1 ? VN / 4 : 1];
#pragma unroll
      for (int k = 0; k + 3 < VN; k += 4) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(
            make_float2(quotient(y[k]), quotient(y[k + 1])), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(
            make_float2(quotient(y[k + 2]), quotient(y[k + 3])), __NV_SATFINITE, __NV_E4M3);
        o[k / 4] = lo | hi << 16;
      }
      if constexpr (VN == 8) __stcs(reinterpret_cast<uint2*>(at), make_uint2(o[0], o[1]));
      else if constexpr (VN == 4) __stcs(reinterpret_cast<uint32_t*>(at), o[0]);
    };
    if constexpr (BLOCK && VN == 1) {
      // 128 columns are four warps side by side: one exchange for all of the row's groups.
      static_assert(TPR % 128 == 0, "groups of whole warps");
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      float y[CPT][VN];
#pragma unroll
      for (int u = 0; u < CPT; ++u) {
        if (u * TPR >= cols) break;
        const float m = warp_redux_max(values(u, y[u]));
        if (lane == 0) group_max[u][warp] = m;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < CPT; ++u) {
        if (u * TPR >= cols) break;
        const float* g = &group_max[u][warp & ~3];
        const float scale = scale_of(fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])));
        const int c = t + u * TPR;
        if (t % 128 == 0 && c < cols) scales[row * ((cols + 127) / 128) + c / 128] = scale;
        put(u, y[u], Quotient(scale));
      }
    } else if constexpr (BLOCK) {
      // The 128 / VN chunks of a group lie in neighbouring lanes (a row of 8 lanes is shorter
      // than a group).
      constexpr int kLanes = 128 / VN < TPR ? 128 / VN : TPR;
#pragma unroll
      for (int u = 0; u < CPT; ++u) {
        const int c = t + u * TPR;
        float y[VN];
        float m = values(u, y);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float scale = scale_of(m);
        if (t % kLanes == 0 && c < chunks && there)
          scales[row * ((cols + 127) / 128) + c * VN / 128] = scale;
        put(u, y, Quotient(scale));
      }
    } else {
      float y[CPT][VN], m = 0.f;
#pragma unroll
      for (int u = 0; u < CPT; ++u) m = fmaxf(m, values(u, y[u]));
      const float scale = scale_of(row_reduce<TPR, true>(m, red[1]));
      if (t == 0 && there) scales[row] = scale;
      const Quotient quotient(scale);
#pragma unroll
      for (int u = 0; u < CPT; ++u) put(u, y[u], quotient);
    }
  }
}

struct FwdArgs {
  const void *x, *r, *w;
  void *y, *q, *h;
  float *scales, *rstd;
  int64_t xs, rs, rows, cols;
  int wd;
  float eps;
};

template <typename T, typename R, bool QUANT, bool BLOCK, int TPR, int CPT,
          int VN = 16 / (int)sizeof(T)>
int launch_rows(const FwdArgs& a, cudaStream_t st) {
  const int64_t grid = (a.rows + fwd_groups(TPR) - 1) / fwd_groups(TPR);
  add_rmsnorm_rows<T, R, VN, TPR, CPT, QUANT, BLOCK><<<(unsigned)grid, TPR <= 32 ? 256 : TPR, 0, st>>>(
      static_cast<const T*>(a.x), a.xs, static_cast<const R*>(a.r), a.rs, a.w, a.wd,
      static_cast<T*>(a.y), static_cast<uint8_t*>(a.q), a.scales, static_cast<R*>(a.h), a.rstd,
      a.rows, (int)a.cols, a.eps);
  return launch_status(QUANT ? "fk_add_rmsnorm_quant" : "fk_add_rmsnorm_fwd");
}

// Whether every row of x, r and the outputs is whole 16-byte chunks.
template <typename T, typename R>
bool rows_of_chunks(const FwdArgs& a) {
  constexpr int VN = 16 / (int)sizeof(T);
  return a.cols % VN == 0 && aligned16(a.x) && a.xs % VN == 0 && aligned16(a.w) &&
         (!a.r || (aligned16(a.r) && a.rs * (int64_t)sizeof(R) % 16 == 0 && aligned16(a.h))) &&
         (!a.y || aligned16(a.y)) && (!a.q || aligned16(a.q)) &&
         a.rows < ((int64_t)1 << 31);
}

// Runs the chunk kernel where the rows allow it (at most 2048 chunks); -1 where they do not.  256
// threads of 2 chunks beat 128 of 4 at 16384 x 4096 bf16 (forward 83.9 against 85.3 us, 8 bits,
// before their quotients were corrected, 75.1 against 77.3); where 128 threads of 3 suffice, they
// hold more rows at a time.
template <typename T, typename R, bool QUANT, bool BLOCK>
int rows_chunked(const FwdArgs& a, cudaStream_t st) {
  if (!rows_of_chunks<T, R>(a)) return -1;
  const int64_t chunks = a.cols / (16 / (int)sizeof(T));
  if (chunks <= 8) return launch_rows<T, R, QUANT, BLOCK, 8, 1>(a, st);
  if (chunks <= 32) return launch_rows<T, R, QUANT, BLOCK, 32, 1>(a, st);
  if (chunks <= 64) return launch_rows<T, R, QUANT, BLOCK, 32, 2>(a, st);
  if (chunks <= 128) return launch_rows<T, R, QUANT, BLOCK, 32, 4>(a, st);
  if (chunks <= 256) return launch_rows<T, R, QUANT, BLOCK, 128, 2>(a, st);
  if (chunks <= 384) return launch_rows<T, R, QUANT, BLOCK, 128, 3>(a, st);
  if (chunks <= 512) return launch_rows<T, R, QUANT, BLOCK, 256, 2>(a, st);
  if (chunks <= 768) return launch_rows<T, R, QUANT, BLOCK, 256, 3>(a, st);
  if (chunks <= 1024) return launch_rows<T, R, QUANT, BLOCK, 256, 4>(a, st);
  if (chunks <= 2048) return launch_rows<T, R, QUANT, BLOCK, 512, 4>(a, st);
  return -1;
}

// The same with single elements, for rows that are not whole chunks; -1 where they are too long.
template <typename T, typename R, bool QUANT, bool BLOCK>
int rows_single(const FwdArgs& a, cudaStream_t st) {
  if (a.rows >= (int64_t)1 << 31) return -1;
  if (a.cols <= 128) return launch_rows<T, R, QUANT, BLOCK, 128, 1, 1>(a, st);
  if (a.cols <= 512) return launch_rows<T, R, QUANT, BLOCK, 128, 4, 1>(a, st);
  if (a.cols <= 1024) return launch_rows<T, R, QUANT, BLOCK, 128, 8, 1>(a, st);
  if (a.cols <= 2048) return launch_rows<T, R, QUANT, BLOCK, 256, 8, 1>(a, st);
  if (a.cols <= 4096) return launch_rows<T, R, QUANT, BLOCK, 512, 8, 1>(a, st);
  if (a.cols <= 8192) return launch_rows<T, R, QUANT, BLOCK, 512, 16, 1>(a, st);
  return -1;
}

// mean(w dy h) s^3, s times three: s^3 by itself leaves the normal range where a row's size is
// beyond 1e12, while the product is of the size of dy / h^2.
__device__ __forceinline__ float times_cube(float mean, float s) { return mean * s * s * s; }

// ------------------------------------------------------------------ backward, chunks ----
// Persistent CTAs, so that dw is summed in registers: a thread has the same columns in every
// row it meets.  Each CTA leaves one partial row of dw; a second kernel adds those up.
struct BwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dr;
  float* part;
  int64_t dys, dhs;
  int rows, cols, wd;
};

// g of one chunk from its dy, h, dh; stores dx (and dr).
template <typename T, typename R, int VN>
__device__ __forceinline__ void bwd_store(const Chunk<T, VN>& dy, const Chunk<R, VN>& h,
                                          const Chunk<R, VN>& dh, const float (&w)[VN], float s,
                                          float c2, bool has_dh, T* dx, R* dr) {
  Chunk<T, VN> ox;
  Chunk<R, VN> orr;
#pragma unroll
  for (int k = 0; k < VN; ++k) {
    float g = s * (w[k] * Elt<T>::to_f(dy.e[k])) - Elt<R>::to_f(h.e[k]) * c2;
    if (has_dh) g += Elt<R>::to_f(dh.e[k]);
    ox.e[k] = Elt<T>::from_f(g);
    orr.e[k] = Elt<R>::from_f(g);
  }
  ox.store(dx);
  if (sizeof(T) != sizeof(R)) orr.store(dr);
}

// Rows of at most 64 chunks: TPR lanes of a warp take a row (no CTA barrier per row), and the
// next row is loaded while this one is worked on.
template <typename T, typename R, int TPR, int CPT>
__global__ void __launch_bounds__(256) add_rmsnorm_bwd_lanes(BwdArgs a) {
  constexpr int VN = 16 / (int)sizeof(T), kGroups = 256 / TPR;
  extern __shared__ float sum[];  // [cols]
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int chunks = a.cols / VN;
  const T* dy = static_cast<const T*>(a.dy);
  const R *dh = static_cast<const R*>(a.dh), *h = static_cast<const R*>(a.h);
  const float inv_cols = 1.0f / (float)a.cols;
  float wv[CPT][VN], acc[CPT][VN];
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = t + u * TPR;
#pragma unroll
    for (int k = 0; k < VN; ++k) wv[u][k] = acc[u][k] = 0.f;
    if (c < chunks) load_weights<VN>(a.w, a.wd, c * VN, wv[u]);
  }
  Chunk<T, VN> ndy[CPT];
  Chunk<R, VN> nh[CPT], ndh[CPT];
  float ns = 0.f;
  auto load = [&](int row) {
    if (row >= a.rows) return;
    ns = __ldg(a.rstd + row);
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = t + u * TPR;
      if (c < chunks) {
        ndy[u].load(dy + row * a.dys + c * VN);
        nh[u].load(h + (int64_t)row * a.cols + c * VN);
        if (dh) ndh[u].load(dh + row * a.dhs + c * VN);
      }
    }
  };
  const int step = gridDim.x * kGroups;
  // Whole warps go round together: a group past the last row only joins the shuffles.
  const int first = blockIdx.x * kGroups + group, warp_first = first - (threadIdx.x & 31) / TPR;
  load(first);
  for (int row = first, wr = warp_first; wr < a.rows; row += step, wr += step) {
    const bool there = row < a.rows;
    Chunk<T, VN> vdy[CPT];
    Chunk<R, VN> vh[CPT], vdh[CPT];
    const float s = ns;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      vdy[u] = ndy[u];
      vh[u] = nh[u];
      vdh[u] = ndh[u];
    }
    load(row + step);
    float dot = 0.f;
#pragma unroll
    for (int u = 0; u < CPT; ++u)
      if (there && t + u * TPR < chunks)
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const float d = Elt<T>::to_f(vdy[u].e[k]), hv = Elt<R>::to_f(vh[u].e[k]);
          dot = fmaf(wv[u][k] * d, hv, dot);
          acc[u][k] = fmaf(d * hv, s, acc[u][k]);
        }
    dot = row_reduce<TPR, false>(dot, nullptr);
    const float c2 = times_cube(dot * inv_cols, s);
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = t + u * TPR;
      if (there && c < chunks)
        bwd_store<T, R, VN>(vdy[u], vh[u], vdh[u], wv[u], s, c2, dh != nullptr,
                            static_cast<T*>(a.dx) + (int64_t)row * a.cols + c * VN,
                            static_cast<R*>(a.dr) + (int64_t)row * a.cols + c * VN);
    }
  }
  for (int c = threadIdx.x; c < a.cols; c += 256) sum[c] = 0.f;
  for (int g = 0; g < kGroups; ++g) {  // the groups' sums, in their order
    __syncthreads();
    if (group == g)
#pragma unroll
      for (int u = 0; u < CPT; ++u) {
        const int c = t + u * TPR;
        if (c < chunks)
#pragma unroll
          for (int k = 0; k < VN; ++k) sum[c * VN + k] += acc[u][k];
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.cols; c += 256)
    a.part[(int64_t)blockIdx.x * a.cols + c] = sum[c];
}

// Longer rows: the CTA takes a row.  Rows of dy, h and dh arrive in a ring of shared-memory stages
// by cp.async.bulk; a stage is refilled as soon as all threads have its chunks in registers, which
// the reduction's barrier tells.  Bound by HBM: 86 us at 16384 x 4096 bf16 (6.3 TB/s), 4 us more
// for dw.  Stages: 3 where they take 72 KB (three CTAs an SM), else 2, or 1.  At 4096 x 16384 bf16
// 96 us for 83 of bytes, 48 bytes spilled; with an fp32 stream a stage is 160 KB, so one CTA an SM
// holds one stage, and 176 bytes are spilled: 212 us for 166.
constexpr int kBwdMaxStages = 3;
template <typename T, typename R, int THREADS, int CPT>
__global__ void __launch_bounds__(THREADS) add_rmsnorm_bwd_ring(BwdArgs a, int stages) {
  constexpr int VN = 16 / (int)sizeof(T);
  using CT = Chunk<T, VN>;
  using CR = Chunk<R, VN>;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) uint64_t full[kBwdMaxStages];
  __shared__ float red[2][32];
  const int tid = threadIdx.x, chunks = a.cols / VN;
  const T* dy = static_cast<const T*>(a.dy);
  const R *dh = static_cast<const R*>(a.dh), *h = static_cast<const R*>(a.h);
  const uint32_t tb = (uint32_t)a.cols * sizeof(T), rb = (uint32_t)a.cols * sizeof(R);
  const uint32_t stage_bytes = tb + (dh ? 2 : 1) * rb;
  const float inv_cols = 1.0f / (float)a.cols;
  float wv[CPT][VN], acc[CPT][VN];
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = tid + u * THREADS;
#pragma unroll
    for (int k = 0; k < VN; ++k) wv[u][k] = acc[u][k] = 0.f;
    if (c < chunks) load_weights<VN>(a.w, a.wd, c * VN, wv[u]);
  }
  auto issue = [&](int row, int q) {
    if (row >= a.rows) return;
    unsigned char* at = ring + q * stage_bytes;
    ptx::fence_proxy_async_smem();
    ptx::mbar_arrive_expect_tx(&full[q], stage_bytes);
    ptx::bulk_g2s(at, dy + row * a.dys, tb, &full[q]);
    ptx::bulk_g2s(at + tb, h + (int64_t)row * a.cols, rb, &full[q]);
    if (dh) ptx::bulk_g2s(at + tb + rb, dh + row * a.dhs, rb, &full[q]);
  };
  const int step = gridDim.x;
  if (tid == 0) {
    for (int q = 0; q < stages; ++q) ptx::mbar_init(&full[q], 1);
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    for (int q = 0; q < stages; ++q) issue(blockIdx.x + q * step, q);
  }
  __syncthreads();
  bool ok = true;
  int q = 0, phase = 0, parity = 0;
  float ns = (int)blockIdx.x < a.rows ? __ldg(a.rstd + blockIdx.x) : 0.f;
  for (int row = blockIdx.x; row < a.rows; row += step) {
    const float s = ns;
    if (row + step < a.rows) ns = __ldg(a.rstd + row + step);
    ok = ptx::mbar_wait(&full[q], (uint32_t)phase, ok ? kPolls : 1u) && ok;
    const unsigned char* at = ring + q * stage_bytes;
    CT vdy[CPT];
    CR vh[CPT], vdh[CPT];
    float dot = 0.f;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = tid + u * THREADS;
      if (c < chunks) {
        vdy[u].u[0] = reinterpret_cast<const uint4*>(at)[c];
#pragma unroll
        for (int i = 0; i < CR::N16; ++i) {
          vh[u].u[i] = reinterpret_cast<const uint4*>(at + tb)[c * CR::N16 + i];
          if (dh) vdh[u].u[i] = reinterpret_cast<const uint4*>(at + tb + rb)[c * CR::N16 + i];
        }
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const float d = Elt<T>::to_f(vdy[u].e[k]), hv = Elt<R>::to_f(vh[u].e[k]);
          dot = fmaf(wv[u][k] * d, hv, dot);
          acc[u][k] = fmaf(d * hv, s, acc[u][k]);
        }
      }
    }
    // (A thread whose wait ran out poisons the row for all of them, and its part of dw below.)
    if (!ok) dot = __int_as_float(0x7fc00000);
    dot = row_reduce<THREADS, false>(dot, red[parity]);  // its barrier frees the stage
    if (tid == 0 && ok) issue(row + stages * step, q);
    const float c2 = times_cube(dot * inv_cols, s);
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = tid + u * THREADS;
      if (c < chunks)
        bwd_store<T, R, VN>(vdy[u], vh[u], vdh[u], wv[u], s, c2, dh != nullptr,
                            static_cast<T*>(a.dx) + (int64_t)row * a.cols + c * VN,
                            static_cast<R*>(a.dr) + (int64_t)row * a.cols + c * VN);
    }
    parity ^= 1;
    if (++q == stages) {
      q = 0;
      phase ^= 1;
    }
  }
  float* prow = a.part + (int64_t)blockIdx.x * a.cols;
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = tid + u * THREADS;
    if (c < chunks)
#pragma unroll
      for (int k = 0; k < VN; k += 4)
        *reinterpret_cast<float4*>(prow + c * VN + k) =
            make_float4(acc[u][k], acc[u][k + 1], acc[u][k + 2], acc[u][k + 3]);
  }
  if (!ok) {  // what came late or not at all is in the sums, and may still be on its way
    for (int c = tid; c < chunks; c += THREADS)
      for (int k = 0; k < VN; ++k) prow[c * VN + k] = __int_as_float(0x7fc00000);
    for (int i = 0; i < 2 * stages; ++i) ptx::mbar_wait(&full[i >> 1], (uint32_t)(i & 1), kPolls);
  }
}

// CTAs of KERNEL that an SM holds, looked up again when the device or the sizes change.
template <auto KERNEL>
int resident_ctas(int threads, int smem) {
  static thread_local int asked_dev = -1, asked_smem, answer;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (asked_dev != dev || asked_smem != smem) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&answer, KERNEL, threads, (size_t)smem) !=
            cudaSuccess ||
        answer < 1) {
      cudaGetLastError();
      answer = 1;
    }
    asked_dev = dev;
    asked_smem = smem;
  }
  return answer < kMaxGridPerSm ? answer : kMaxGridPerSm;
}

template <typename T, typename R, int TPR, int CPT>
int launch_bwd_lanes(const BwdArgs& a, int* grid, cudaStream_t st) {
  constexpr auto kern = add_rmsnorm_bwd_lanes<T, R, TPR, CPT>;
  const int smem = a.cols * 4, groups = 256 / TPR;
  const int most = num_sms() * resident_ctas<kern>(256, smem);
  const int want = (a.rows + groups - 1) / groups;
  *grid = want < most ? want : most;
  kern<<<*grid, 256, smem, st>>>(a);
  return launch_status("fk_add_rmsnorm_bwd");
}

template <typename T, typename R, int THREADS, int CPT>
int launch_bwd_ring(const BwdArgs& a, int* grid, cudaStream_t st) {
  constexpr auto kern = add_rmsnorm_bwd_ring<T, R, THREADS, CPT>;
  allow_shared_memory<kern>(1024);
  const int stage = a.cols * ((int)sizeof(T) + (a.dh ? 2 : 1) * (int)sizeof(R));
  constexpr int kMost = 224 * 1024;  // of a CTA
  if (stage > kMost) return -1;
  int stages = 72 * 1024 / stage;
  stages = stages >= 3 ? 3 : 2 * stage <= kMost ? 2 : 1;
  const int smem = stages * stage;
  const int most = num_sms() * resident_ctas<kern>(THREADS, smem);
  *grid = a.rows < most ? a.rows : most;
  kern<<<*grid, THREADS, smem, st>>>(a, stages);
  return launch_status("fk_add_rmsnorm_bwd");
}

// Runs a chunk kernel where the rows allow it; -1 where they do not.
template <typename T, typename R>
int bwd_chunked(const BwdArgs& a, int* grid, cudaStream_t st) {
  constexpr int VN = 16 / (int)sizeof(T);
  const bool fits = a.cols % VN == 0 && aligned16(a.dy) && a.dys % VN == 0 && aligned16(a.h) &&
                    (!a.dh || (aligned16(a.dh) && a.dhs * (int64_t)sizeof(R) % 16 == 0)) &&
                    aligned16(a.w) && aligned16(a.dx) && aligned16(a.dr);
  if (!fits) return -1;
  const int chunks = a.cols / VN;
  if (chunks <= 8) return launch_bwd_lanes<T, R, 8, 1>(a, grid, st);
  if (chunks <= 32) return launch_bwd_lanes<T, R, 32, 1>(a, grid, st);
  if (chunks <= 64) return launch_bwd_lanes<T, R, 32, 2>(a, grid, st);
  if (chunks <= 256) return launch_bwd_ring<T, R, 128, 2>(a, grid, st);
  if (chunks <= 512) return launch_bwd_ring<T, R, 256, 2>(a, grid, st);
  if (chunks <= 1024) return launch_bwd_ring<T, R, 512, 2>(a, grid, st);
  if (chunks <= 2048) return launch_bwd_ring<T, R, 1024, 2>(a, grid, st);
  return -1;
}

// ------------------------------------------------------------------ backward, columns ---
// Rows of any width, stride and alignment: thread t of the CTA has the columns t, t + THREADS,
// ... as single elements, the next row's on their way while this one is worked on.  22 us at
// 5003 x 1111 bf16 with an fp32 residual (element loops 54, tiles through shared memory 40).  Above
// 4096 columns 208 to 268 bytes are spilled: 90 us at 4096 x 8191 bf16 for 42 of bytes.
template <typename T, typename R, int THREADS, int CPT>
__global__ void __launch_bounds__(THREADS) add_rmsnorm_bwd_columns(BwdArgs a) {
  __shared__ float red[2][32];
  const int t = threadIdx.x;
  const T* dy = static_cast<const T*>(a.dy);
  const R *dh = static_cast<const R*>(a.dh), *h = static_cast<const R*>(a.h);
  const float inv_cols = 1.0f / (float)a.cols;
  float wv[CPT], acc[CPT];
  T ndy[CPT];
  R nh[CPT], ndh[CPT];
  float ns = 0.f;
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = t + u * THREADS;
    acc[u] = 0.f;
    wv[u] = c < a.cols ? load_wd(a.w, a.wd, c) : 0.f;
    ndy[u] = Elt<T>::from_f(0.f);
    nh[u] = ndh[u] = Elt<R>::from_f(0.f);
  }
  auto load = [&](int row) {
    if (row >= a.rows) return;
    ns = __ldg(a.rstd + row);
    const T* pd = dy + row * a.dys;
    const R *ph = h + (int64_t)row * a.cols, *pg = dh + row * a.dhs;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = t + u * THREADS;
      if (c < a.cols) {
        ndy[u] = pd[c];
        nh[u] = ph[c];
        if (dh) ndh[u] = pg[c];
      }
    }
  };
  const int step = gridDim.x;
  int parity = 0;
  load(blockIdx.x);
  for (int row = blockIdx.x; row < a.rows; row += step, parity ^= 1) {
    const float s = ns;
    float d[CPT], hv[CPT], g[CPT], dot = 0.f;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      d[u] = Elt<T>::to_f(ndy[u]);
      hv[u] = Elt<R>::to_f(nh[u]);
      g[u] = Elt<R>::to_f(ndh[u]);
      dot = fmaf(wv[u] * d[u], hv[u], dot);
      acc[u] = fmaf(d[u] * hv[u], s, acc[u]);
    }
    load(row + step);
    dot = row_reduce<THREADS, false>(dot, red[parity]);
    const float c2 = times_cube(dot * inv_cols, s);
    T* px = static_cast<T*>(a.dx) + (int64_t)row * a.cols;
    R* pr = static_cast<R*>(a.dr) + (int64_t)row * a.cols;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int c = t + u * THREADS;
      if (c < a.cols) {
        const float v = s * (wv[u] * d[u]) - hv[u] * c2 + g[u];
        px[c] = Elt<T>::from_f(v);
        if (sizeof(T) != sizeof(R)) pr[c] = Elt<R>::from_f(v);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < CPT; ++u) {
    const int c = t + u * THREADS;
    if (c < a.cols) a.part[(int64_t)blockIdx.x * a.cols + c] = acc[u];
  }
}

template <typename T, typename R, int THREADS, int CPT>
int launch_bwd_columns(const BwdArgs& a, int* grid, cudaStream_t st) {
  constexpr auto kern = add_rmsnorm_bwd_columns<T, R, THREADS, CPT>;
  const int most = num_sms() * resident_ctas<kern>(THREADS, 0);
  *grid = a.rows < most ? a.rows : most;
  kern<<<*grid, THREADS, 0, st>>>(a);
  return launch_status("fk_add_rmsnorm_bwd");
}

template <typename T, typename R>
int bwd_columns(const BwdArgs& a, int* grid, cudaStream_t st) {
  if (a.cols <= 128) return launch_bwd_columns<T, R, 128, 1>(a, grid, st);
  if (a.cols <= 512) return launch_bwd_columns<T, R, 128, 4>(a, grid, st);
  if (a.cols <= 1024) return launch_bwd_columns<T, R, 128, 8>(a, grid, st);
  if (a.cols <= 2048) return launch_bwd_columns<T, R, 256, 8>(a, grid, st);
  if (a.cols <= 4096) return launch_bwd_columns<T, R, 512, 8>(a, grid, st);
  if (a.cols <= 8192) return launch_bwd_columns<T, R, 512, 16>(a, grid, st);
  return -1;
}

// ------------------------------------------------------------------ any shape -----------
// One CTA per row, element loops.  h is re-read by the thread that wrote it.  At 1677 x 40000 bf16
// forward 277 us, backward 651 and 47 for dw, for 83 of bytes each; in 8 bits 392 per row and 906
// per 128 columns for 73.
template <typename T, typename R>
__global__ void __launch_bounds__(256) add_rmsnorm_fwd_generic(
    const T* __restrict__ x, int64_t xs, const R* __restrict__ r, int64_t rs,
    const void* __restrict__ w, int wd, T* __restrict__ y, R* h, float* __restrict__ rstd,
    int64_t rows, int64_t cols, float eps) {
  __shared__ float red[32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const R hv = Elt<R>::from_f(Elt<T>::to_f(x[row * xs + c]) + Elt<R>::to_f(r[row * rs + c]));
      h[row * cols + c] = hv;
      const float f = Elt<R>::to_f(hv);
      ss = fmaf(f, f, ss);
    }
    const float s = rsqrtf(block_sum(ss, red) / (float)cols + eps);
    if (threadIdx.x == 0 && rstd) rstd[row] = s;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x)
      y[row * cols + c] = Elt<T>::from_f(Elt<R>::to_f(h[row * cols + c]) * s * load_wd(w, wd, c));
  }
}

template <typename T, typename R>
__global__ void __launch_bounds__(256) add_rmsnorm_bwd_generic(
    const T* __restrict__ dy, int64_t dys, const R* __restrict__ dh, int64_t dhs,
    const R* __restrict__ h, const void* __restrict__ w, int wd, const float* __restrict__ rstd,
    T* __restrict__ dx, R* __restrict__ dr, float* __restrict__ part, int64_t rows,
    int64_t cols) {
  __shared__ float red[32];
  float* prow = part + (int64_t)blockIdx.x * cols;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) prow[c] = 0.f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float s = rstd[row];
    float dot = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = Elt<T>::to_f(dy[row * dys + c]), hv = Elt<R>::to_f(h[row * cols + c]);
      dot = fmaf(load_wd(w, wd, c) * d, hv, dot);
      prow[c] = fmaf(d * hv, s, prow[c]);  // each column is one thread's
    }
    const float c2 = times_cube(block_sum(dot, red) / (float)cols, s);
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = Elt<T>::to_f(dy[row * dys + c]), hv = Elt<R>::to_f(h[row * cols + c]);
      float g = s * (load_wd(w, wd, c) * d) - hv * c2;
      if (dh) g += Elt<R>::to_f(dh[row * dhs + c]);
      dx[row * cols + c] = Elt<T>::from_f(g);
      if (dr) dr[row * cols + c] = Elt<R>::from_f(g);
    }
  }
}

// r == nullptr: h is x itself and is not written.
template <typename T, typename R>
__global__ void __launch_bounds__(256) add_rmsnorm_quant_generic(
    const T* __restrict__ x, int64_t xs, const R* __restrict__ r, int64_t rs,
    const void* __restrict__ w, int wd, uint8_t* __restrict__ q, float* __restrict__ scales,
    R* h, int64_t rows, int64_t cols, int64_t block, float eps) {
  __shared__ float red[32];
  const int64_t groups = (cols + block - 1) / block;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float f = Elt<T>::to_f(x[row * xs + c]);
      if (r) {
        const R hv = Elt<R>::from_f(f + Elt<R>::to_f(r[row * rs + c]));
        h[row * cols + c] = hv;
        f = Elt<R>::to_f(hv);
      }
      ss = fmaf(f, f, ss);
    }
    const float s = rsqrtf(block_sum(ss, red) / (float)cols + eps);
    __syncthreads();  // the groups below read columns that other threads wrote
    auto value = [&](int64_t c) {
      const float f = r ? Elt<R>::to_f(h[row * cols + c]) : Elt<T>::to_f(x[row * xs + c]);
      return f * s * load_wd(w, wd, c);
    };
    for (int64_t g = 0; g < groups; ++g) {
      const int64_t c0 = g * block, c1 = c0 + block < cols ? c0 + block : cols;
      float m = 0.f;
      for (int64_t c = c0 + threadIdx.x; c < c1; c += blockDim.x) m = fmaxf(m, fabsf(value(c)));
      const float scale = scale_of(block_max(m, red));
      if (threadIdx.x == 0) scales[row * groups + g] = scale;
      for (int64_t c = c0 + threadIdx.x; c < c1; c += blockDim.x)
        q[row * cols + c] = to_e4m3(value(c) / scale);
    }
  }
}

// dw[c] = sum over the G partial rows in a fixed order, cast to W.  One CTA of 32 warps per
// 32 columns: warp w sums partial rows w, w+32, ..., the warp sums are added in warp order.
template <typename W>
__global__ void __launch_bounds__(1024) add_rmsnorm_dw_reduce(const float* __restrict__ part,
                                                              int G, int64_t cols,
                                                              W* __restrict__ dw) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int g = warp; g < G; g += 32) s += part[(int64_t)g * cols + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += red[i][lane];
    dw[c] = Elt<W>::from_f(t);
  }
}

inline int row_grid(int64_t rows) {
  const int64_t g = (int64_t)num_sms() * kMaxGridPerSm;
  return (int)(rows < g ? rows : g);
}
inline size_t bwd_ws_bytes(int64_t rows, int64_t cols) {
  return (size_t)row_grid(rows) * (size_t)cols * sizeof(float);
}

template <typename T, typename R>
int fwd_t(const void* x, int64_t xs, const void* r, int64_t rs, const void* w, int wd, void* y,
          void* h, float* rstd, int64_t rows, int64_t cols, float eps, cudaStream_t st) {
  const FwdArgs a{x, r, w, y, nullptr, h, nullptr, rstd, xs, rs, rows, cols, wd, eps};
  int done = rows_chunked<T, R, false, false>(a, st);
  if (done < 0) done = rows_single<T, R, false, false>(a, st);
  if (done >= 0) return done;
  add_rmsnorm_fwd_generic<T, R><<<row_grid(rows), 256, 0, st>>>(
      static_cast<const T*>(x), xs, static_cast<const R*>(r), rs, w, wd, static_cast<T*>(y),
      static_cast<R*>(h), rstd, rows, cols, eps);
  return launch_status("fk_add_rmsnorm_fwd");
}

template <typename T, typename R>
int bwd_t(const void* dy, int64_t dys, const void* dh, int64_t dhs, const void* h, const void* w,
          int wd, const float* rstd, void* dx, void* dr, float* part, int64_t rows, int64_t cols,
          int* grid, cudaStream_t st) {
  if (rows < ((int64_t)1 << 31) - (1 << 20) && cols < (1 << 20)) {
    const BwdArgs a{dy,  dh,  h,         w,         rstd, dx, dr,
                    part, dys, dhs, (int)rows, (int)cols, wd};
    int done = bwd_chunked<T, R>(a, grid, st);
    if (done < 0) done = bwd_columns<T, R>(a, grid, st);
    if (done >= 0) return done;
  }
  *grid = row_grid(rows);
  add_rmsnorm_bwd_generic<T, R><<<*grid, 256, 0, st>>>(
      static_cast<const T*>(dy), dys, static_cast<const R*>(dh), dhs, static_cast<const R*>(h), w,
      wd, rstd, static_cast<T*>(dx), static_cast<R*>(dr), part, rows, cols);
  return launch_status("fk_add_rmsnorm_bwd");
}

template <typename T, typename R>
int quant_t(const void* x, int64_t xs, const void* r, int64_t rs, const void* w, int wd, void* q,
            float* scales, void* h, int64_t rows, int64_t cols, int64_t block, float eps,
            cudaStream_t st) {
  const FwdArgs a{x, r, w, nullptr, q, h, scales, nullptr, xs, rs, rows, cols, wd, eps};
  int done = block == cols ? rows_chunked<T, R, true, false>(a, st)
                           : rows_chunked<T, R, true, true>(a, st);
  if (done < 0)
    done = block == cols ? rows_single<T, R, true, false>(a, st)
                         : rows_single<T, R, true, true>(a, st);
  if (done >= 0) return done;
  add_rmsnorm_quant_generic<T, R><<<row_grid(rows), 256, 0, st>>>(
      static_cast<const T*>(x), xs, static_cast<const R*>(r), rs, w, wd,
      static_cast<uint8_t*>(q), scales, static_cast<R*>(h), rows, cols, block, eps);
  return launch_status("fk_add_rmsnorm_quant");
}

}  // namespace
}  // namespace fk

// Binds T (dtype) and R (the residual's type: dtype or FK_F32).
#define FK_DISPATCH_TR(dtype, r_dtype, ...)                                  \
  FK_DISPATCH_DTYPE(dtype, {                                                 \
    if ((r_dtype) == (dtype)) { using res_t = scalar_t; __VA_ARGS__; }       \
    else { using res_t = float; __VA_ARGS__; }                               \
  })

extern "C" int fk_add_rmsnorm_fwd(const void* x, int64_t x_row_stride, const void* r,
                                  int64_t r_row_stride, int r_dtype, const void* weight,
                                  int w_dtype, void* y, void* h, float* rstd, int64_t rows,
                                  int64_t cols, float eps, int dtype, void* stream) {
  FK_CHECK_ARG(rows >= 0 && cols >= 1, "fk_add_rmsnorm_fwd: bad shape [%lld, %lld]",
               (long long)rows, (long long)cols);
  FK_CHECK_ARG(fk::valid_dtype(dtype) && fk::valid_dtype(w_dtype), "fk_add_rmsnorm_fwd: bad dtype");
  FK_CHECK_ARG(r_dtype == dtype || r_dtype == FK_F32,
               "fk_add_rmsnorm_fwd: the residual has x's type or fp32");
  FK_CHECK_ARG(x_row_stride >= cols && r_row_stride >= cols,
               "fk_add_rmsnorm_fwd: row stride < cols");
  if (rows == 0) return FK_OK;
  FK_CHECK_ARG(x && r && weight && y && h, "fk_add_rmsnorm_fwd: null pointer");
  FK_DISPATCH_TR(dtype, r_dtype, return (fk::fwd_t<scalar_t, res_t>(
                                     x, x_row_stride, r, r_row_stride, weight, w_dtype, y, h, rstd,
                                     rows, cols, eps, fk::as_stream(stream))));
  return FK_OK;
}

extern "C" int fk_add_rmsnorm_bwd_workspace_size(int64_t rows, int64_t cols, size_t* bytes) {
  FK_CHECK_ARG(bytes != nullptr, "fk_add_rmsnorm_bwd_workspace_size: null output");
  FK_CHECK_ARG(rows >= 0 && cols >= 1, "fk_add_rmsnorm_bwd_workspace_size: bad shape");
  *bytes = rows == 0 ? 0 : fk::bwd_ws_bytes(rows, cols);
  return FK_OK;
}

extern "C" int fk_add_rmsnorm_bwd(const void* dy, int64_t dy_row_stride, const void* dh,
                                  int64_t dh_row_stride, const void* h, int r_dtype,
                                  const void* weight, int w_dtype, const float* rstd, void* dx,
                                  void* dr, void* dw, void* workspace, size_t workspace_bytes,
                                  int64_t rows, int64_t cols, int dtype, void* stream) {
  FK_CHECK_ARG(rows >= 0 && cols >= 1, "fk_add_rmsnorm_bwd: bad shape [%lld, %lld]",
               (long long)rows, (long long)cols);
  FK_CHECK_ARG(fk::valid_dtype(dtype) && fk::valid_dtype(w_dtype), "fk_add_rmsnorm_bwd: bad dtype");
  FK_CHECK_ARG(r_dtype == dtype || r_dtype == FK_F32,
               "fk_add_rmsnorm_bwd: the residual has x's type or fp32");
  FK_CHECK_ARG(dw && weight, "fk_add_rmsnorm_bwd: null pointer");
  cudaStream_t st = fk::as_stream(stream);
  if (rows == 0) {
    cudaMemsetAsync(dw, 0, (size_t)cols * fk::dtype_size(w_dtype), st);
    return fk::launch_status("fk_add_rmsnorm_bwd(zero dw)");
  }
  FK_CHECK_ARG(dy && h && rstd && dx, "fk_add_rmsnorm_bwd: null pointer");
  FK_CHECK_ARG(dr || r_dtype == dtype, "fk_add_rmsnorm_bwd: dr is needed where the types differ");
  FK_CHECK_ARG(dy_row_stride >= cols && (!dh || dh_row_stride >= cols),
               "fk_add_rmsnorm_bwd: row stride < cols");
  const size_t need = fk::bwd_ws_bytes(rows, cols);
  if (workspace == nullptr || workspace_bytes < need || !fk::aligned16(workspace))
    return fk::fail(FK_ERR_WORKSPACE,
                    "fk_add_rmsnorm_bwd: need %zu aligned workspace bytes, got %zu", need,
                    workspace_bytes);
  float* part = static_cast<float*>(workspace);
  int grid = 0, s = FK_OK;
  FK_DISPATCH_TR(dtype, r_dtype, s = (fk::bwd_t<scalar_t, res_t>(
                                     dy, dy_row_stride, dh, dh_row_stride, h, weight, w_dtype,
                                     rstd, dx, r_dtype == dtype ? nullptr : dr, part, rows, cols,
                                     &grid, st)));
  if (s != FK_OK) return s;
  const unsigned rgrid = (unsigned)((cols + 31) / 32);
  FK_DISPATCH_DTYPE(w_dtype, (fk::add_rmsnorm_dw_reduce<scalar_t><<<rgrid, 1024, 0, st>>>(
                                 part, grid, cols, static_cast<scalar_t*>(dw))));
  return fk::launch_status("fk_add_rmsnorm_bwd(dw reduce)");
}

extern "C" int fk_add_rmsnorm_quant(const void* x, int64_t x_row_stride, const void* r,
                                    int64_t r_row_stride, int r_dtype, const void* weight,
                                    int w_dtype, void* q, float* scales, void* h, int64_t rows,
                                    int64_t cols, int64_t block, float eps, int dtype,
                                    void* stream) {
  FK_CHECK_ARG(rows >= 0 && cols >= 1, "fk_add_rmsnorm_quant: bad shape [%lld, %lld]",
               (long long)rows, (long long)cols);
  FK_CHECK_ARG(fk::valid_dtype(dtype) && fk::valid_dtype(w_dtype),
               "fk_add_rmsnorm_quant: bad dtype");
  FK_CHECK_ARG(r_dtype == dtype || r_dtype == FK_F32,
               "fk_add_rmsnorm_quant: the residual has x's type or fp32");
  FK_CHECK_ARG(block == 0 || block == 128, "fk_add_rmsnorm_quant: block is 0 (the row) or 128");
  FK_CHECK_ARG(x_row_stride >= cols && (!r || r_row_stride >= cols),
               "fk_add_rmsnorm_quant: row stride < cols");
  if (rows == 0) return FK_OK;
  FK_CHECK_ARG(x && weight && q && scales, "fk_add_rmsnorm_quant: null pointer");
  FK_CHECK_ARG(!r || h, "fk_add_rmsnorm_quant: h is needed with a residual");
  FK_DISPATCH_TR(dtype, r_dtype, return (fk::quant_t<scalar_t, res_t>(
                                     x, x_row_stride, r, r_row_stride, weight, w_dtype, q, scales,
                                     h, rows, cols, block ? block : cols, eps,
                                     fk::as_stream(stream))));
  return FK_OK;
}
