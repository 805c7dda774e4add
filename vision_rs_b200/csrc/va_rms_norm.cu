// Root-mean-square norm with the residual's addition, forward and backward:
//
//   h = x + res,   r = 1/√(mean(h²) + eps),   y = h·r·w          per row
//
// y in the input's type, or in 8 bits (e4m3): y ≈ q·s with s = max|y| / 448
// over a row, or over each `group` columns of it.  Backward, with g = dy·w:
//
//   dh = r·(g − h·r²·mean(g·h)) + grad_h,    dw = Σ_rows dy·h·r
//
// (dh is the gradient of x and of res alike; grad_h is the gradient that
// arrives at h itself along the residual).
//
// Bound: HBM.  Each row is read once and lives in registers between the
// reduction and the output: TPR threads own a row, each NV vectors of 16
// bytes.  All arithmetic and sums are f32; the forward norm uses the f32 sum
// h, not the rounded h that it stores.  The weight gradient is a sum over rows: each
// block walks its rows with the columns' sums in registers and writes one
// partial row; a second kernel adds the partials in a fixed order, so the
// result does not depend on scheduling (no atomics).
//
// Measured (B200): 16384 × 4096 bf16 to 8 bits 75–78 µs (0.93–0.95 of the copy
// rate; 128 × 4 or 512 × 1 threads and vectors a row instead of 256 × 2: 105,
// 101 µs); 25616 × 384 f32 60 µs for the pair (launch list: 21, 26 and 5).
#include <cuda_fp8.h>

#include <type_traits>

#include "va_common.cuh"
#include "va_psa.h"

namespace va {
namespace {

constexpr float kE4M3Max = 448.0f;
constexpr float kSmallestAmax = 7.8886090522101181e-31f;  // 2^-100: a row of zeros gets a scale that is not zero

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
  static constexpr float none = 0.0f;
};
struct Max {
  static __device__ __forceinline__ float of(float a, float b) { return max_nan(a, b); }
  static constexpr float none = 0.0f;  // of absolute values
};

template <typename OP> __device__ __forceinline__ float warp_all(float v, int lanes = 32) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = OP::of(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Over the TPR threads of a row (a warp, or the whole block).  `buf`: 32 floats
// of its own for each call site, so one barrier a call is enough until the
// caller's next barrier.
template <typename OP, int TPR> __device__ __forceinline__ float row_all(float v, float* buf) {
  v = warp_all<OP>(v);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < TPR / 32 ? buf[threadIdx.x & 31] : OP::none;
    v = warp_all<OP>(v);
  }
  return v;
}

// 8 bits: y/s needs no r (y = h·w·r, s = max|y|/448), so the row's h·w is scaled by 448 / max|h·w| directly: two
// roundings an element less, each of which can tip a value over to the next of the 8-bit grid.
struct Quant {
  float amax, mul;  // max|y|, and what h·w is multiplied by
};
__device__ __forceinline__ Quant quant_of(float top, float r) {  // top: max|h·w|
  const float y = top * r, amax = max_nan(y, kSmallestAmax);
  return {amax, y >= kSmallestAmax ? kE4M3Max / top : r * (kE4M3Max / amax)};
}

struct NormArgs {
  const void *x, *res, *w;
  void *h, *y;
  uint8_t* q;
  float* scale;
  int w_f32;
  long long rows;
  int cols, group;
  float eps;
};

template <typename T, int N>
__device__ __forceinline__ void load_w(const void* w, int w_f32, int c, float (&o)[N]) {
  if (w_f32) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w) + c + j));
      o[j] = f.x, o[j + 1] = f.y, o[j + 2] = f.z, o[j + 3] = f.w;
    }
  } else {
    Bytes16<T>::get(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c)), o);
  }
}

__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
      " mov.b32 %0, {lo, hi};\n}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ float max_nan_abs(float a, float b) {  // max(a, |b|), NaN if either is
  float d;
  asm("{\n .reg .f32 t;\n abs.f32 t, %2;\n max.NaN.f32 %0, %1, t;\n}" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint8_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

constexpr int rows_per_block(int tpr) { return tpr == 32 ? 8 : 1; }
constexpr int block_threads(int tpr) { return tpr == 32 ? 256 : tpr; }

template <typename T, int TPR, int NV, bool F8>
__global__ void __launch_bounds__(block_threads(TPR)) rms_norm_kernel(NormArgs a) {
  using B = Bytes16<T>;
  constexpr int VEC = B::N;
  __shared__ float red[2][32];
  const long long row = (long long)blockIdx.x * rows_per_block(TPR) + (TPR == 32 ? threadIdx.x >> 5 : 0);
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x, nvec = a.cols / VEC;
  if (row >= a.rows) return;  // TPR = 32 only: whole warps
  const long long base = row * a.cols;
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + base);
  const uint4* res = reinterpret_cast<const uint4*>(static_cast<const T*>(a.res) + base);
  const bool with_res = a.res != nullptr;
  float v[NV][VEC], ss = 0.0f;
  uint4 vx[NV], vr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * TPR;
    if (c < nvec) {
      vx[i] = x[c];
      if (with_res) vr[i] = res[c];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * TPR;
    if (c < nvec) {
      B::get(vx[i], v[i]);
      if (with_res) {
        float r[VEC];
        B::get(vr[i], r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += r[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss = fmaf(v[i][j], v[i][j], ss);
      if (a.h) reinterpret_cast<uint4*>(static_cast<T*>(a.h) + base)[c] = B::put(v[i]);
    }
  }
  ss = row_all<Sum, TPR>(ss, red[0]);
  const float r = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * TPR;
    if (c < nvec) {
      float w[VEC];
      load_w<T>(a.w, a.w_f32, c * VEC, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (F8) {
          v[i][j] *= w[j];
          top = max_nan_abs(top, v[i][j]);
        } else {
          v[i][j] = v[i][j] * r * w[j];
        }
      }
      if constexpr (!F8) reinterpret_cast<uint4*>(static_cast<T*>(a.y) + base)[c] = B::put(v[i]);
    }
  }
  if constexpr (F8) {
    const bool whole = a.group == a.cols;
    Quant z{};
    if (whole) {
      z = quant_of(row_all<Max, TPR>(top, red[1]), r);
      if (t == 0) a.scale[row] = z.amax / kE4M3Max;
    }
    const int lanes = a.group / VEC;  // of one group (a power of two ≤ 32 unless the group is the row)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * TPR;
      if (!whole) {
        float m = 0.0f;
        if (c < nvec) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) m = max_nan_abs(m, v[i][j]);
        }
        z = quant_of(warp_all<Max>(m, lanes), r);
        if (c < nvec && (t & (lanes - 1)) == 0) a.scale[row * (a.cols / a.group) + c / lanes] = z.amax / kE4M3Max;
      }
      if (c < nvec) {
        const float inv = z.mul;
        uint32_t q[VEC / 4];
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          q[j / 4] = to_e4m3x4(v[i][j] * inv, v[i][j + 1] * inv, v[i][j + 2] * inv, v[i][j + 3] * inv);
        if constexpr (VEC == 8) reinterpret_cast<uint2*>(a.q + base)[c] = make_uint2(q[0], q[1]);
        else reinterpret_cast<uint32_t*>(a.q + base)[c] = q[0];
      }
    }
  }
}

// Any width, alignment and group: one block a row, columns read again for each pass.
template <typename T, bool F8>
__global__ void __launch_bounds__(256) rms_norm_any_kernel(NormArgs a) {
  __shared__ float red[2][32];
  const long long row = blockIdx.x, base = row * a.cols;
  const T *x = static_cast<const T*>(a.x) + base, *res = a.res ? static_cast<const T*>(a.res) + base : nullptr;
  auto at = [&](int c) { return to_f32(x[c]) + (res ? to_f32(res[c]) : 0.0f); };
  auto weight = [&](int c) {
    return a.w_f32 ? static_cast<const float*>(a.w)[c] : to_f32(static_cast<const T*>(a.w)[c]);
  };
  float ss = 0.0f;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float v = at(c);
    ss = fmaf(v, v, ss);
  }
  ss = row_all<Sum, 256>(ss, red[0]);
  const float r = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
  if constexpr (F8) {
    const bool whole = a.group == a.cols;
    if (whole) {
      float top = 0.0f;
      for (int c = threadIdx.x; c < a.cols; c += 256) top = max_nan_abs(top, at(c) * weight(c));
      const Quant z = quant_of(row_all<Max, 256>(top, red[1]), r);
      if (threadIdx.x == 0) a.scale[row] = z.amax / kE4M3Max;
      for (int c = threadIdx.x; c < a.cols; c += 256) a.q[base + c] = to_e4m3(at(c) * weight(c) * z.mul);
    } else {
      const int ng = a.cols / a.group, lane = threadIdx.x & 31;
      for (int g = threadIdx.x >> 5; g < ng; g += 8) {  // a warp for each group
        float m = 0.0f;
        for (int c = lane; c < a.group; c += 32) m = max_nan_abs(m, at(g * a.group + c) * weight(g * a.group + c));
        const Quant z = quant_of(warp_all<Max>(m), r);
        if (lane == 0) a.scale[row * ng + g] = z.amax / kE4M3Max;
        for (int c = g * a.group + lane; c < (g + 1) * a.group; c += 32) a.q[base + c] = to_e4m3(at(c) * weight(c) * z.mul);
      }
    }
  }
  __syncthreads();  // h may be x or res itself: every thread has read the row before any of it is written
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float v = at(c);
    if (a.h) static_cast<T*>(a.h)[base + c] = from_f32<T>(v);
    if constexpr (!F8) static_cast<T*>(a.y)[base + c] = from_f32<T>(v * r * weight(c));
  }
}

struct NormBwdArgs {
  const void *dy, *h, *w, *grad_h;
  void* dh;
  float* partial;  // [gridDim.x][cols]
  int w_f32;
  long long rows;
  int cols;
  float eps;
};

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(block_threads(TPR)) rms_norm_bwd_kernel(NormBwdArgs a) {
  using B = Bytes16<T>;
  constexpr int VEC = B::N, RPB = rows_per_block(TPR);
  __shared__ float red[4][32];
  extern __shared__ float wsum[];  // TPR = 32: [8][cols], the warps' column sums
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x, nvec = a.cols / VEC;
  const int sub = TPR == 32 ? threadIdx.x >> 5 : 0;
  const bool with_gh = a.grad_h != nullptr;
  let_next_start();
  float dw[NV][VEC] = {}, w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t + i * TPR < nvec) load_w<T>(a.w, a.w_f32, (t + i * TPR) * VEC, w[i]);
  int turn = 0;
  for (long long row = (long long)blockIdx.x * RPB + sub; row < a.rows; row += (long long)gridDim.x * RPB) {
    const long long base = row * a.cols;
    const uint4* pdy = reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + base);
    const uint4* ph = reinterpret_cast<const uint4*>(static_cast<const T*>(a.h) + base);
    const uint4* pg = reinterpret_cast<const uint4*>(static_cast<const T*>(a.grad_h) + base);
    uint4 dy[NV], h[NV], gh[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * TPR;
      if (c < nvec) {
        dy[i] = pdy[c];
        h[i] = ph[c];
        if (with_gh) gh[i] = pg[c];
      }
    }
    float ss = 0.0f, sg = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * TPR < nvec) {
        float fd[VEC], fh[VEC];
        B::get(dy[i], fd);
        B::get(h[i], fh);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ss = fmaf(fh[j], fh[j], ss);
          sg = fmaf(fd[j] * w[i][j], fh[j], sg);
        }
      }
    // the two buffers alternate, so a row's reduction never meets the previous row's readers
    ss = row_all<Sum, TPR>(ss, red[turn]);
    sg = row_all<Sum, TPR>(sg, red[turn + 1]);
    turn ^= 2;
    const float r = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
    const float k = r * r * (sg / (float)a.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * TPR;
      if (c < nvec) {
        float fd[VEC], fh[VEC], o[VEC];
        B::get(dy[i], fd);
        B::get(h[i], fh);
        if (with_gh) B::get(gh[i], o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float g = r * (fd[j] * w[i][j] - fh[j] * k);
          o[j] = with_gh ? o[j] + g : g;
          dw[i][j] = fmaf(fd[j], fh[j] * r, dw[i][j]);
        }
        reinterpret_cast<uint4*>(static_cast<T*>(a.dh) + base)[c] = B::put(o);
      }
    }
  }
  float* out = a.partial + (long long)blockIdx.x * a.cols;
  if constexpr (TPR == 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * TPR < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) wsum[sub * a.cols + (t + i * TPR) * VEC + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      float s = 0.0f;
      for (int k = 0; k < 8; ++k) s += wsum[k * a.cols + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * TPR < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[(t + i * TPR) * VEC + j] = dw[i][j];
  }
}

// Any width and alignment: the block's column sums live in its partial row.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_bwd_any_kernel(NormBwdArgs a) {
  __shared__ float red[4][32];
  float* out = a.partial + (long long)blockIdx.x * a.cols;
  for (int c = threadIdx.x; c < a.cols; c += 256) out[c] = 0.0f;  // read and written by this thread alone
  auto weight = [&](int c) {
    return a.w_f32 ? static_cast<const float*>(a.w)[c] : to_f32(static_cast<const T*>(a.w)[c]);
  };
  int turn = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const long long base = row * a.cols;
    const T *dy = static_cast<const T*>(a.dy) + base, *h = static_cast<const T*>(a.h) + base;
    float ss = 0.0f, sg = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float fh = to_f32(h[c]);
      ss = fmaf(fh, fh, ss);
      sg = fmaf(to_f32(dy[c]) * weight(c), fh, sg);
    }
    ss = row_all<Sum, 256>(ss, red[turn]);
    sg = row_all<Sum, 256>(sg, red[turn + 1]);
    turn ^= 2;
    const float r = 1.0f / sqrtf(ss / (float)a.cols + a.eps), k = r * r * (sg / (float)a.cols);
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float fh = to_f32(h[c]), fd = to_f32(dy[c]);
      out[c] = fmaf(fd, fh * r, out[c]);
      const float g = a.grad_h ? to_f32(static_cast<const T*>(a.grad_h)[base + c]) : 0.0f;
      static_cast<T*>(a.dh)[base + c] = from_f32<T>(r * (fd * weight(c) - fh * k) + g);
    }
  }
}

// dw[c] = Σ partial[p][c]: 32 rows of 32 threads, each its rows p ≡ ty (mod 32) in order, then the 32 in order.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ partial, float* __restrict__ dw,
                                                          int n, int cols) {
  __shared__ float s[32][33];
  wait_for_previous();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
  float v = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = ty; p < n; p += 32) v += partial[(long long)p * cols + c];
  }
  s[ty][tx] = v;
  __syncthreads();
  v = warp_all<Sum>(s[tx][ty]);  // column ty's 32 sums
  if (tx == 0 && blockIdx.x * 32 + ty < cols) dw[blockIdx.x * 32 + ty] = v;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Threads for each row and vectors for each thread; tpr 0: only the any-width kernel takes it.
struct NormShape {
  int tpr, nv;
};
NormShape norm_shape(long long rows, int nvec) {
  // Many rows: few threads a row, up to four vectors each (more loads in flight a thread, cheaper
  // reductions).  Few rows (under two blocks an SM): one vector a thread, the row's latency counts.
  const int most = rows <= 296 ? 1 : 4;
  for (int tpr : {32, 256, 512, 1024})
    if (nvec <= tpr * most) return {tpr, (nvec + tpr - 1) / tpr};
  return nvec <= 4096 ? NormShape{1024, (nvec + 1023) / 1024} : NormShape{0, 0};
}

template <typename F> int with_shape(NormShape s, F&& f) {
  auto nv = [&](auto tpr) -> int {
    if (s.nv <= 1) return f(tpr, std::integral_constant<int, 1>{});
    if (s.nv == 2) return f(tpr, std::integral_constant<int, 2>{});
    return f(tpr, std::integral_constant<int, 4>{});
  };
  switch (s.tpr) {
    case 32: return nv(std::integral_constant<int, 32>{});
    case 256: return nv(std::integral_constant<int, 256>{});
    case 512: return nv(std::integral_constant<int, 512>{});
    default: return nv(std::integral_constant<int, 1024>{});
  }
}

int check_norm(long long rows, int cols, float eps) {
  VA_CHECK_ARG(rows >= 0 && rows < (1LL << 31) && cols > 0, "rms_norm: %lld rows of %d columns", rows, cols);
  VA_CHECK_ARG(eps >= 0.0f, "rms_norm: eps must not be negative");
  return VA_OK;
}

template <typename T, bool F8> int rms_norm(NormArgs a, cudaStream_t st) {
  if (int rc = check_norm(a.rows, a.cols, a.eps)) return rc;
  if (a.group == 0) a.group = a.cols;
  VA_CHECK_ARG(a.group > 0 && a.cols % a.group == 0, "rms_norm: %d columns in groups of %d", a.cols, a.group);
  if (a.rows == 0) return VA_OK;
  VA_CHECK_ARG(a.x && a.w && (F8 ? a.q && a.scale : a.y != nullptr), "rms_norm: null pointer");
  constexpr int VEC = 16 / sizeof(T);
  const int lanes = a.group / VEC;
  const bool vec = a.cols % VEC == 0 && aligned16(a.x) && aligned16(a.res) && aligned16(a.w) && aligned16(a.h) &&
                   (F8 ? aligned16(a.q) : aligned16(a.y)) &&
                   (a.group == a.cols || (a.group % VEC == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0));
  const NormShape s = vec ? norm_shape(a.rows, a.cols / VEC) : NormShape{0, 0};
  if (s.tpr == 0) {
    rms_norm_any_kernel<T, F8><<<(unsigned)a.rows, 256, 0, st>>>(a);
    return check_launch("rms_norm");
  }
  return with_shape(s, [&](auto tpr, auto nv) -> int {
    constexpr int R = rows_per_block(tpr);
    rms_norm_kernel<T, tpr, nv, F8><<<(unsigned)((a.rows + R - 1) / R), block_threads(tpr), 0, st>>>(a);
    return check_launch("rms_norm");
  });
}

// Partial rows of the weight gradient: a function of the sizes alone, so that the order of its sums is too.
int bwd_blocks(long long rows, int cols) {
  const long long want = 148LL * (cols <= 1024 ? 4 : 8);
  return (int)std::max(1LL, std::min(want, cols <= 1024 ? (rows + 7) / 8 : rows));
}

template <typename T> int rms_norm_bwd(NormBwdArgs a, float* dw, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (int rc = check_norm(a.rows, a.cols, a.eps)) return rc;
  VA_CHECK_ARG(dw && (a.rows == 0 || (a.dy && a.h && a.w && a.dh)), "rms_norm backward: null pointer");
  const int nb = bwd_blocks(a.rows, a.cols);
  const size_t need = (size_t)nb * a.cols * 4;
  if (!ws || ws_bytes < need)
    return set_error(VA_ERR_WORKSPACE, "rms_norm backward: workspace %zu < %zu bytes", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) & 15)
    return set_error(VA_ERR_ALIGN, "rms_norm backward: workspace needs 16-byte alignment");
  if (a.rows == 0) {  // no row to read, w neither: it may be null
    const cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)a.cols * 4, st);
    return e == cudaSuccess ? VA_OK : set_error(VA_ERR_LAUNCH, "rms_norm backward: %s", cudaGetErrorString(e));
  }
  a.partial = static_cast<float*>(ws);
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = a.cols % VEC == 0 && aligned16(a.dy) && aligned16(a.h) && aligned16(a.w) && aligned16(a.grad_h) &&
                   aligned16(a.dh);
  const int nvec = a.cols / VEC;
  auto go = [&](auto kernel, int threads, size_t smem) -> int {
    kernel<<<nb, threads, smem, st>>>(a);
    return check_launch("rms_norm backward");
  };
  // A warp a row up to 128 vectors; wider rows take a block, at most four vectors a thread beside the
  // columns' sums (a 16-bit row of 8192 columns: 512 threads x 2).
  const size_t sums = (size_t)8 * a.cols * 4;  // of the block's eight rows, <= 32 KB
  int rc;
  if (!vec || nvec > 2048) rc = go(rms_norm_bwd_any_kernel<T>, 256, 0);
  else if (nvec <= 32) rc = go(rms_norm_bwd_kernel<T, 32, 1>, 256, sums);
  else if (nvec <= 64) rc = go(rms_norm_bwd_kernel<T, 32, 2>, 256, sums);
  else if (nvec <= 128) rc = go(rms_norm_bwd_kernel<T, 32, 4>, 256, sums);
  else if (nvec <= 256) rc = go(rms_norm_bwd_kernel<T, 128, 2>, 128, 0);
  else if (nvec <= 512) rc = go(rms_norm_bwd_kernel<T, 512, 1>, 512, 0);
  else if (nvec <= 1024) rc = go(rms_norm_bwd_kernel<T, 512, 2>, 512, 0);
  else rc = go(rms_norm_bwd_kernel<T, 512, 4>, 512, 0);
  if (rc) return rc;
  return launch_behind("rms_norm weight gradient", column_sum_kernel, (a.cols + 31) / 32, 1024, 0, st, a.partial, dw, nb,
                       a.cols);
}

}  // namespace
}  // namespace va

using namespace va;

#define VA_RMS_NORM_ENTRIES(sfx, CT, T)                                                                              \
  int va_rms_norm_fwd_##sfx(const CT* x, const CT* residual, const void* w, int w_is_f32, CT* h, CT* y,              \
                            long long rows, int cols, float eps, va_stream_t stream) {                               \
    NormArgs a{x, residual, w, h, y, nullptr, nullptr, w_is_f32, rows, cols, 0, eps};                                \
    return rms_norm<T, false>(a, (cudaStream_t)stream);                                                              \
  }                                                                                                                  \
  int va_rms_norm_fwd_f8_##sfx(const CT* x, const CT* residual, const void* w, int w_is_f32, CT* h, uint8_t* q,      \
                               float* scale, long long rows, int cols, int group, float eps, va_stream_t stream) {   \
    NormArgs a{x, residual, w, h, nullptr, q, scale, w_is_f32, rows, cols, group, eps};                              \
    return rms_norm<T, true>(a, (cudaStream_t)stream);                                                               \
  }                                                                                                                  \
  int va_rms_norm_bwd_##sfx(const CT* dy, const CT* h, const void* w, int w_is_f32, const CT* grad_h, CT* dh,        \
                            float* dw, long long rows, int cols, float eps, void* workspace, size_t ws_bytes,        \
                            va_stream_t stream) {                                                                    \
    NormBwdArgs a{dy, h, w, grad_h, dh, nullptr, w_is_f32, rows, cols, eps};                                         \
    return rms_norm_bwd<T>(a, dw, workspace, ws_bytes, (cudaStream_t)stream);                                        \
  }

extern "C" {
size_t va_rms_norm_bwd_workspace_bytes(long long rows, int cols) {
  if (rows < 0 || cols <= 0) return 0;
  return align256((size_t)bwd_blocks(rows, cols) * cols * 4);
}
VA_RMS_NORM_ENTRIES(bf16, va_bf16, __nv_bfloat16)
VA_RMS_NORM_ENTRIES(f16, void, __half)
VA_RMS_NORM_ENTRIES(f32, float, float)
}  // extern "C"
