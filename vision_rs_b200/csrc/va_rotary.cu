// Rotary positions: every pair (a, b) of a head's first `rot` dimensions turns
// by the angle θ = position · inv_freq[i],
//
//   a' = c·(a·cos θ − b·sin θ),   b' = c·(a·sin θ + b·cos θ),
//
// with pairs (x[2i], x[2i+1]) (interleaved) or (x[i], x[i + rot/2]) (halves);
// dimensions from `rot` on are copied.  The map is c times a rotation, so the
// gradient goes back through the same map with −θ (`backward`).
//
// The angle is reduced in 64 bits: a position of 10^5 times a frequency of
// 1 rad leaves only ~7 bits of fraction in f32 (0.008 rad), while the
// remainder in turns, position · inv_freq / 2π − nearest integer, is exact to
// 10^-11 in f64 and goes on in f32 (sincospif).
//
// Bound: HBM, each element read and written once.  A block owns a few tokens:
// it computes their rot/2 (cos, sin) pairs once into shared memory, and its
// threads then walk (token, head) rows with 16-byte accesses, all q and k
// heads of a token in the same block, so the sines cost 1/heads of a pair
// each.  One launch serves q and k.
#include <cuda_fp16.h>

#include "va_common.cuh"

namespace va {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxTokensPerBlock = 4;
constexpr int kMaxRot = 512;

template <typename T> struct RotCvt;
template <> struct RotCvt<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct RotCvt<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct RotCvt<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

template <typename T, int P> struct alignas(sizeof(T) * P) Pack {
  T v[P];
};

struct RotTensor {
  const void* in;
  void* out;
  long long in_row, in_head, out_row, out_head;  // strides in elements
  int heads;
};

// P pairs (or P copied elements) per thread and row; P·sizeof(T) ≤ 16.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads)
rotary_kernel(RotTensor q, RotTensor k, const void* __restrict__ positions, int pos64,
              const double* __restrict__ inv_freq, int tokens, int tpb, int dim, int rot, float factor,
              float sin_sign) {
  __shared__ float2 cs[kMaxTokensPerBlock * (kMaxRot / 2)];
  const int half = rot / 2, t0 = blockIdx.x * tpb, nt = min(tpb, tokens - t0);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthreads = blockDim.x * blockDim.y;
  for (int i = tid; i < nt * half; i += nthreads) {
    const int t = i / half, f = i - t * half;
    const double pos = pos64 ? (double)static_cast<const long long*>(positions)[t0 + t]
                             : (double)static_cast<const int*>(positions)[t0 + t];
    const double turns = pos * (inv_freq[f] * 0.15915494309189533577);  // 1 / 2π
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(factor * c, sin_sign * factor * s);
  }
  __syncthreads();

  using V = Pack<T, P>;
  const int heads = q.heads + k.heads, nrot = half / P, nchunk = nrot + (dim - rot) / P;
  for (int c = threadIdx.x; c < nchunk; c += blockDim.x) {
#pragma unroll 2
    for (int r = threadIdx.y; r < nt * heads; r += blockDim.y) {
      const int t = r / heads, h = r - t * heads;
      const bool is_q = h < q.heads;
      const RotTensor& x = is_q ? q : k;
      const int hx = is_q ? h : h - q.heads;
      const T* in = static_cast<const T*>(x.in) + (t0 + t) * x.in_row + hx * x.in_head;
      T* out = static_cast<T*>(x.out) + (t0 + t) * x.out_row + hx * x.out_head;
      if (c >= nrot) {
        const int d = rot + (c - nrot) * P;
        *reinterpret_cast<V*>(out + d) = *reinterpret_cast<const V*>(in + d);
        continue;
      }
      const int ia = INTERLEAVED ? 2 * P * c : P * c, ib = INTERLEAVED ? ia + P : ia + half;
      V a = *reinterpret_cast<const V*>(in + ia), b = *reinterpret_cast<const V*>(in + ib);
      const float2* w = cs + t * half + c * P;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        // the pair's two elements: a[i], b[i], or (interleaved) neighbours of the 2P elements (a, b)
        T& ta = INTERLEAVED ? (2 * i < P ? a.v[(2 * i) % P] : b.v[(2 * i) % P]) : a.v[i];
        T& tb = INTERLEAVED ? (2 * i + 1 < P ? a.v[(2 * i + 1) % P] : b.v[(2 * i + 1) % P]) : b.v[i];
        const float fa = RotCvt<T>::to(ta), fb = RotCvt<T>::to(tb);
        const float2 z = w[i];
        ta = RotCvt<T>::from(fa * z.x - fb * z.y);
        tb = RotCvt<T>::from(fa * z.y + fb * z.x);
      }
      *reinterpret_cast<V*>(out + ia) = a;
      *reinterpret_cast<V*>(out + ib) = b;
    }
  }
}

// Largest P ∈ {16 bytes, …, 1 element} that divides every offset an access starts at.
int pick_pack(const RotTensor* x, int n, int elem, int dim, int rot) {
  for (int p = 16 / elem; p > 1; p /= 2) {
    bool ok = (rot / 2) % p == 0 && (dim - rot) % p == 0;
    for (int i = 0; i < n && ok; ++i) {
      const RotTensor& t = x[i];
      ok = (reinterpret_cast<uintptr_t>(t.in) | reinterpret_cast<uintptr_t>(t.out)) % (p * elem) == 0 &&
           (t.in_row % p) == 0 && (t.in_head % p) == 0 && (t.out_row % p) == 0 && (t.out_head % p) == 0;
    }
    if (ok) return p;
  }
  return 1;
}

template <typename T>
int rotary(RotTensor q, RotTensor k, const void* positions, int position_bytes, const double* inv_freq, int tokens,
           int dim, int rot, int interleaved, int backward, float factor, cudaStream_t st) {
  VA_CHECK_ARG(tokens >= 0 && dim > 0 && rot >= 0 && rot <= dim && rot % 2 == 0 && rot <= kMaxRot,
               "rotary: %d tokens, head size %d, %d rotated dimensions (even, at most the head size and %d)", tokens,
               dim, rot, kMaxRot);
  VA_CHECK_ARG(q.heads > 0 && k.heads >= 0 && q.heads + k.heads <= 65535, "rotary: %d query and %d key heads",
               q.heads, k.heads);
  VA_CHECK_ARG(position_bytes == 4 || position_bytes == 8, "rotary: positions of %d bytes", position_bytes);
  if (tokens == 0) return VA_OK;
  VA_CHECK_ARG(q.in && q.out && (k.heads == 0 || (k.in && k.out)) && positions && (rot == 0 || inv_freq),
               "rotary: null pointer");
  if (k.heads == 0) k = RotTensor{q.in, q.out, 0, 0, 0, 0, 0};
  const RotTensor both[2] = {q, k};
  const int p = pick_pack(both, k.heads ? 2 : 1, (int)sizeof(T), dim, rot);
  const int nchunk = rot / 2 / p + (dim - rot) / p;
  const int bx = std::min(nchunk, kRotThreads), by = kRotThreads / bx;
  // several tokens a block once there are blocks enough for every SM (the sines of a token cost one pass anyway)
  const int tpb = tokens >= 148 * 8 * kMaxTokensPerBlock ? kMaxTokensPerBlock : tokens >= 148 * 16 ? 2 : 1;
  const dim3 block(bx, by), grid((tokens + tpb - 1) / tpb);
  auto go = [&](auto kernel) -> int {
    kernel<<<grid, block, 0, st>>>(q, k, positions, position_bytes == 8, inv_freq, tokens, tpb, dim, rot, factor,
                                   backward ? -1.0f : 1.0f);
    return check_launch("rotary");
  };
  switch (p) {
    case 8:
      if constexpr (sizeof(T) == 2) return interleaved ? go(rotary_kernel<T, 8, true>) : go(rotary_kernel<T, 8, false>);
    case 4: return interleaved ? go(rotary_kernel<T, 4, true>) : go(rotary_kernel<T, 4, false>);
    case 2: return interleaved ? go(rotary_kernel<T, 2, true>) : go(rotary_kernel<T, 2, false>);
    default: return interleaved ? go(rotary_kernel<T, 1, true>) : go(rotary_kernel<T, 1, false>);
  }
}

}  // namespace
}  // namespace va

using namespace va;

#define VA_ROTARY_ENTRY(name, CT, T)                                                                                \
  int name(const CT* q, const CT* k, CT* q_out, CT* k_out, const int64_t* strides, const void* positions,           \
           int position_bytes, const double* inv_freq, int tokens, int num_heads, int num_kv_heads, int head_dim,   \
           int rot_dim, int interleaved, int backward, float factor, va_stream_t stream) {                          \
    if (!strides) return set_error(VA_ERR_SHAPE, "rotary: null pointer");                                           \
    const RotTensor tq{q, q_out, strides[0], strides[1], strides[4], strides[5], num_heads};                        \
    const RotTensor tk{k, k_out, strides[2], strides[3], strides[6], strides[7], num_kv_heads};                     \
    return rotary<T>(tq, tk, positions, position_bytes, inv_freq, tokens, head_dim, rot_dim, interleaved, backward, \
                     factor, (cudaStream_t)stream);                                                                 \
  }

extern "C" {
VA_ROTARY_ENTRY(va_rotary_bf16, va_bf16, __nv_bfloat16)
VA_ROTARY_ENTRY(va_rotary_f16, void, __half)
VA_ROTARY_ENTRY(va_rotary_f32, float, float)
}  // extern "C"
