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
// Bound: HBM, each element read and written once.  A block owns one or a few
// tokens: it computes their rot/2 (cos, sin) pairs once into shared memory,
// and a thread keeps those of its chunk in registers over the heads that it
// turns with 16-byte accesses, all q and k heads of a token in the same block.
// One launch serves q and k.  Measured (B200): 16384 tokens, 32 + 8 heads of
// 128, 64 rotated, f16, 63–65 µs = 0.8 of the copy rate (two heads in flight a
// thread instead of six: 85 µs; pairs read from shared memory for each head: 95).
#include "va_common.cuh"

namespace va {
namespace {

constexpr int kRotThreads = 256;
constexpr int kBatch = 6;         // heads of a thread that are in flight together
constexpr int kMaxAngles = 2048;  // of a block (16 KB)
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

// P elements ↔ f32 (16 bytes at once, or one by one).
template <typename T, int P> __device__ __forceinline__ void widen(const Pack<T, P>& v, float (&f)[P]) {
  if constexpr (sizeof(T) * P == 16) {
    Bytes16<T>::get(*reinterpret_cast<const uint4*>(&v), f);
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) f[i] = RotCvt<T>::to(v.v[i]);
  }
}
template <typename T, int P> __device__ __forceinline__ Pack<T, P> narrow(const float (&f)[P]) {
  Pack<T, P> v;
  if constexpr (sizeof(T) * P == 16) {
    *reinterpret_cast<uint4*>(&v) = Bytes16<T>::put(f);
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) v.v[i] = RotCvt<T>::from(f[i]);
  }
  return v;
}

// P pairs (or P copied elements) per thread and row; P·sizeof(T) ≤ 16.
// Threads: x walks a head's chunks, y the heads, z the block's tokens, so a
// thread's (cos, sin) pairs stay in registers over its heads.  Its first
// kBatch heads are read before the angles are computed: the loads do not
// depend on them, and the angles' latency hides theirs.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads)
rotary_kernel(RotTensor q, RotTensor k, const void* __restrict__ positions, int pos64,
              const double* __restrict__ inv_freq, int tokens, int dim, int rot, float factor, float sin_sign) {
  extern __shared__ float2 cs[];  // [tokens of the block][rot / 2]
  using V = Pack<T, P>;
  const int half = rot / 2, t0 = blockIdx.x * blockDim.z, t = t0 + threadIdx.z, nt = min((int)blockDim.z, tokens - t0);
  const int tid = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x;
  const int nthreads = blockDim.x * blockDim.y * blockDim.z;
  const int heads = t < tokens ? q.heads + k.heads : 0, nrot = half / P, nchunk = nrot + (dim - rot) / P;
  const T *q_in = static_cast<const T*>(q.in) + t * q.in_row, *k_in = static_cast<const T*>(k.in) + t * k.in_row;
  T *q_out = static_cast<T*>(q.out) + t * q.out_row, *k_out = static_cast<T*>(k.out) + t * k.out_row;
  auto in_of = [&](int h) { return h < q.heads ? q_in + h * q.in_head : k_in + (h - q.heads) * k.in_head; };
  auto out_of = [&](int h) { return h < q.heads ? q_out + h * q.out_head : k_out + (h - q.heads) * k.out_head; };
  // the chunk's first and second vector (a copied chunk has only the first)
  auto at = [&](int c, int& ia, int& ib) {
    ia = c >= nrot ? rot + (c - nrot) * P : INTERLEAVED ? 2 * P * c : P * c;
    ib = INTERLEAVED ? ia + P : ia + half;
  };
  auto turn = [&](V& a, V& b, const float2 (&w)[P]) {
    float fa[P], fb[P];
    widen<T, P>(a, fa);
    widen<T, P>(b, fb);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      // the pair's two elements: a[i], b[i], or (interleaved) neighbours of the 2P elements (a, b)
      float& xa = INTERLEAVED ? (2 * i < P ? fa[(2 * i) % P] : fb[(2 * i) % P]) : fa[i];
      float& xb = INTERLEAVED ? (2 * i + 1 < P ? fa[(2 * i + 1) % P] : fb[(2 * i + 1) % P]) : fb[i];
      const float ya = xa * w[i].x - xb * w[i].y, yb = xa * w[i].y + xb * w[i].x;
      xa = ya;
      xb = yb;
    }
    a = narrow<T, P>(fa);
    b = narrow<T, P>(fb);
  };

  V va[kBatch], vb[kBatch];
  const int c0 = threadIdx.x;  // < nchunk
  int ia, ib;
  at(c0, ia, ib);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int h = threadIdx.y + i * blockDim.y;
    if (h < heads) {
      const T* in = in_of(h);
      va[i] = *reinterpret_cast<const V*>(in + ia);
      if (c0 < nrot) vb[i] = *reinterpret_cast<const V*>(in + ib);
    }
  }
  for (int i = tid; i < nt * half; i += nthreads) {
    const int ti = i / half, f = i - ti * half;
    const double pos = pos64 ? (double)static_cast<const long long*>(positions)[t0 + ti]
                             : (double)static_cast<const int*>(positions)[t0 + ti];
    const double turns = pos * (inv_freq[f] * 0.15915494309189533577);  // 1 / 2π
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(factor * c, sin_sign * factor * s);
  }
  __syncthreads();
  float2 w[P];
  auto angles = [&](int c) {
    if (c < nrot) {
#pragma unroll
      for (int i = 0; i < P; ++i) w[i] = cs[threadIdx.z * half + c * P + i];
    }
  };
  angles(c0);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int h = threadIdx.y + i * blockDim.y;
    if (h < heads) {
      T* out = out_of(h);
      if (c0 < nrot) {
        turn(va[i], vb[i], w);
        *reinterpret_cast<V*>(out + ib) = vb[i];
      }
      *reinterpret_cast<V*>(out + ia) = va[i];
    }
  }
  // what is left: more heads than a batch, heads of more chunks than threads
  for (int c = c0; c < nchunk; c += blockDim.x) {
    if (c > c0) {
      at(c, ia, ib);
      angles(c);
    }
    for (int h = threadIdx.y + (c == c0 ? kBatch * blockDim.y : 0); h < heads; h += blockDim.y) {
      const T* in = in_of(h);
      T* out = out_of(h);
      V a = *reinterpret_cast<const V*>(in + ia);
      if (c < nrot) {
        V b = *reinterpret_cast<const V*>(in + ib);
        turn(a, b, w);
        *reinterpret_cast<V*>(out + ib) = b;
      }
      *reinterpret_cast<V*>(out + ia) = a;
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
  // A batch of heads a thread where there are tokens enough to fill the SMs with such blocks, else one; tokens fill
  // what is left of a block (their angles fit its shared memory).
  const int heads = q.heads + k.heads, bx = std::min(nchunk, kRotThreads);
  const int per_thread = tokens >= 148 * 8 ? kBatch : 1;
  const int by = std::max(1, std::min(kRotThreads / bx, (heads + per_thread - 1) / per_thread));
  const int bz = std::max(1, std::min(std::min(kRotThreads / (bx * by), kMaxAngles / std::max(rot / 2, 1)),
                                      std::min(64, ceil_div(tokens, 148 * 4))));
  const dim3 block(bx, by, bz), grid(ceil_div(tokens, bz));
  const size_t smem = (size_t)bz * (rot / 2) * sizeof(float2);
  auto go = [&](auto kernel) -> int {
    kernel<<<grid, block, smem, st>>>(q, k, positions, position_bytes == 8, inv_freq, tokens, dim, rot, factor,
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
