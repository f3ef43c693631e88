// K12 -- distillation from a teacher's top logits: loss and gradient.
//
// Per row, with temperature T, the student's logits x over the whole
// vocabulary and K kept teacher logits t_j at columns i_j:
//   p = softmax(t / T) over the kept entries,  q = softmax(x / T)
//   loss  = w T^2 sum_j p_j (log p_j - log q[i_j])
//   dx_i  = w T (q_i - sum of p_j with i_j = i)
// An entry with a negative column is absent.  A row without weight (w = 0) or
// without a kept entry gives zeros whatever it holds.
//
// HBM-bound: the loss reads the row once (an online maximum and sum of
// exponentials), the gradient reads it again (mostly from L2) and writes it
// once.  One block per row.  The exponentials are 2^((x - max) c), c =
// log2(e) / T: the difference first, so that logits near the maximum lose
// nothing and a mask of the type's lowest value does not overflow.  The row's
// sum is float32 per thread and joined in a fixed order; the K terms, and the
// logarithms, are in float64, because the loss is a difference of logarithms
// of size ~10.  The kept columns are
// corrected after the row is written, each by one thread, duplicates summed,
// so nothing depends on an order of atomics.

#include <type_traits>

#include "rowtypes.cuh"

namespace mr {
namespace {

constexpr int kDistThreads = 512;
constexpr int kDistUnroll = 4;
constexpr int kDistMaxK = 256;

struct DistShared {
  double sum[kDistThreads / 32];
  float top[kDistThreads / 32], part[kDistThreads / 32];
  double p[kDistMaxK];
  float x[kDistMaxK];
  int64_t col[kDistMaxK];
  int bad, kept;
};

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block, to every thread.
__device__ double block_add(double v, double* part) {
  v = warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kDistThreads / 32; ++i) s += part[i];
  return s;
}

__device__ float block_top(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = part[0];
#pragma unroll
  for (int i = 1; i < kDistThreads / 32; ++i) s = fmaxf(s, part[i]);
  return s;
}

// (max, sum of exponentials relative to it) of one thread's values.
struct Online {
  float m = -INFINITY, s = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], float c) {
    float top = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
    if (top > m) {
      s *= exp2f((m - top) * c);
      m = top;
    }
    // nothing but -inf so far: no finite reference to take exponents from
    if (m == -INFINITY) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (f[i] != f[i]) s = f[i];  // a NaN stays
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2f((f[i] - m) * c);
  }
};

template <typename T>
struct RowSpan {
  int head, vecs, loose;
  const uint4* body;
  __device__ __forceinline__ RowSpan(const T* row, int n) {
    constexpr int kN = Vec16<T>::kN;
    const int off = int((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    head = min(n, off ? kN - off : 0);
    vecs = (n - head) / kN;
    loose = n - vecs * kN;
    body = reinterpret_cast<const uint4*>(row + head);
  }
  // the i-th column outside the vectors
  __device__ __forceinline__ int loose_col(int i) const {
    return i < head ? i : i + vecs * Vec16<T>::kN;
  }
};

struct GradOut {
  void* grad;      // the logits' type, or
  uint16_t* hi;    // a bf16 pair
  uint16_t* lo;
};

template <typename T>
__device__ __forceinline__ void put_one(const GradOut& o, int64_t at, float g) {
  if (o.grad) {
    static_cast<T*>(o.grad)[at] = from_f32<T>(g);
  } else {
    const uint16_t h = f32_to_bf16(g);
    o.hi[at] = h;
    o.lo[at] = f32_to_bf16(__fsub_rn(g, bf16_to_f32(h)));
  }
}

template <typename T>
__device__ __forceinline__ void put_vec(const GradOut& o, int64_t at, bool wide,
                                        const float (&g)[Vec16<T>::kN]) {
  constexpr int kN = Vec16<T>::kN;
  if (wide && o.grad) {
    Vec16<T> v;
    v.put(g);
    *reinterpret_cast<uint4*>(static_cast<T*>(o.grad) + at) = v.raw;
  } else if (wide) {
    uint32_t h[kN / 2], l[kN / 2];
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const uint16_t h0 = f32_to_bf16(g[2 * i]), h1 = f32_to_bf16(g[2 * i + 1]);
      h[i] = uint32_t(h0) | (uint32_t(h1) << 16);
      l[i] = uint32_t(f32_to_bf16(__fsub_rn(g[2 * i], bf16_to_f32(h0)))) |
             (uint32_t(f32_to_bf16(__fsub_rn(g[2 * i + 1], bf16_to_f32(h1)))) << 16);
    }
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      reinterpret_cast<uint2*>(o.hi + at)[i] = make_uint2(h[2 * i], h[2 * i + 1]);
      reinterpret_cast<uint2*>(o.lo + at)[i] = make_uint2(l[2 * i], l[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) put_one<T>(o, at + i, g[i]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kDistThreads, 2)
    distill_kernel(const T* logits /* may be the gradient's own storage */, int64_t ld, int n,
                   const float* __restrict__ t_logits, const int64_t* __restrict__ t_index, int k,
                   double temperature, const float* __restrict__ weight, float* __restrict__ loss,
                   const GradOut out, int64_t ldg) {
  __shared__ DistShared sh;
  constexpr int kN = Vec16<T>::kN;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T* row = logits + r * ld;
  const bool want_grad = out.grad || out.hi;
  const RowSpan<T> span(row, n);
  // stores as wide as the loads where the gradient's row lies as the logits' does
  const int64_t g0 = r * ldg;
  bool wide;
  if (out.grad)
    wide = ((reinterpret_cast<uintptr_t>(static_cast<T*>(out.grad) + g0 + span.head)) & 15u) == 0;
  else
    wide = ((reinterpret_cast<uintptr_t>(out.hi + g0 + span.head) |
             reinterpret_cast<uintptr_t>(out.lo + g0 + span.head)) & 7u) == 0;
  if (tid == 0) sh.bad = 0;
  __syncthreads();
  // the teacher's distribution
  const float w = weight ? weight[r] : 1.f;
  float t = -INFINITY;
  if (tid < k) {
    const int64_t col = t_index[r * k + tid];
    sh.col[tid] = col;
    if (col >= n) sh.bad = 1;
    if (col >= 0 && col < n) {
      t = t_logits[r * k + tid];
      sh.x[tid] = to_f32(row[col]);
    }
  }
  const float t_top = block_top(t, sh.top);
  const bool nan_t = __syncthreads_or(tid < k && t != t);
  if (w == 0.f || (t_top == -INFINITY && !nan_t && !sh.bad)) {  // block-uniform
    if (tid == 0 && loss) loss[r] = 0.f;
    if (want_grad) {
      float zero[kN] = {};
      for (int i = tid; i < span.vecs; i += kDistThreads)
        put_vec<T>(out, g0 + span.head + int64_t(i) * kN, wide, zero);
      if (tid < span.loose) put_one<T>(out, g0 + span.loose_col(tid), 0.f);
    }
    return;
  }
  double p = t == -INFINITY ? 0.0 : exp((double(t) - double(t_top)) / temperature);
  const double p_sum = block_add(p, sh.sum);
  const double log_p = (double(t) - double(t_top)) / temperature - log(p_sum);
  p /= p_sum;
  if (tid < k) sh.p[tid] = p;

  // the student's maximum and sum of exponentials
  const float c = float(1.4426950408889634 / temperature);
  Online on;
  if (tid < span.loose) {
    const float f[1] = {to_f32(row[span.loose_col(tid)])};
    on.add(f, c);
  }
  for (int i = tid; i < span.vecs; i += kDistThreads * kDistUnroll) {
    Vec16<T> v[kDistUnroll];
#pragma unroll
    for (int u = 0; u < kDistUnroll; ++u)
      if (i + u * kDistThreads < span.vecs) v[u].raw = span.body[i + u * kDistThreads];
#pragma unroll
    for (int u = 0; u < kDistUnroll; ++u) {
      if (i + u * kDistThreads < span.vecs) {
        float f[kN];
        v[u].get(f);
        on.add(f, c);
      }
    }
  }
  const float top = block_top(on.m, sh.top);
  const double total =
      block_add(on.m == -INFINITY ? double(on.s)
                                  : double(on.s) * double(exp2f((on.m - top) * c)),
                sh.sum);
  const float nan = __int_as_float(0x7fffffff);
  const bool bad = sh.bad != 0;
  if (loss) {
    double term = 0.0;
    if (tid < k && p > 0.0) {
      const double log_q = 0.69314718055994530942 *
                           ((double(sh.x[tid]) - double(top)) * double(c) - log2(total));
      term = p * (log_p - log_q);
    } else if (tid < k && p != p) {
      term = p;
    }
    const double kl = block_add(term, sh.sum);
    if (tid == 0) loss[r] = bad ? nan : float(double(w) * temperature * temperature * kl);
  }
  if (!want_grad) return;
  const float scale = bad ? nan : float(double(w) * temperature);
  const float norm = float(double(scale) / total);
  __syncthreads();  // every thread has read what the gradient may overwrite
  for (int i = tid; i < span.vecs; i += kDistThreads * kDistUnroll) {
    Vec16<T> v[kDistUnroll];
#pragma unroll
    for (int u = 0; u < kDistUnroll; ++u)
      if (i + u * kDistThreads < span.vecs) v[u].raw = span.body[i + u * kDistThreads];
#pragma unroll
    for (int u = 0; u < kDistUnroll; ++u) {
      if (i + u * kDistThreads < span.vecs) {
        float f[kN];
        v[u].get(f);
#pragma unroll
        for (int j = 0; j < kN; ++j) f[j] = exp2f((f[j] - top) * c) * norm;
        put_vec<T>(out, g0 + span.head + int64_t(i + u * kDistThreads) * kN, wide, f);
      }
    }
  }
  if (tid < span.loose) {
    const int col = span.loose_col(tid);
    put_one<T>(out, g0 + col, exp2f((to_f32(row[col]) - top) * c) * norm);
  }
  __syncthreads();  // the kept columns' corrections follow the row
  if (tid < k && sh.col[tid] >= 0 && sh.col[tid] < n) {
    const int64_t col = sh.col[tid];
    double mass = 0.0;
    bool first = true;
    for (int j = 0; j < k; ++j) {
      if (sh.col[j] != col) continue;
      if (j < tid) first = false;
      mass += sh.p[j];
    }
    if (first) {
      const double q = double(exp2f((sh.x[tid] - top) * c)) / total;
      put_one<T>(out, g0 + col, float((q - mass) * double(scale)));
    }
  }
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" int mr_distill_topk(const void* logits, int64_t rows, int n, int64_t ld, int dtype,
                               const float* t_logits, const int64_t* t_index, int k,
                               double temperature, const float* weight, float* loss, void* grad,
                               uint16_t* grad_hi, uint16_t* grad_lo, int64_t ldg, void* stream) {
  if (!logits || !t_logits || !t_index || rows <= 0 || rows > 0x7fffffff || n <= 0 || ld < n ||
      k <= 0 || k > kDistMaxK || !known_dtype(dtype) || !(temperature > 0.0) ||
      !(temperature < 1e30))
    return MR_ERR_ARGUMENT;
  if ((grad_hi == nullptr) != (grad_lo == nullptr) || (grad && grad_hi) ||
      (!loss && !grad && !grad_hi) || ((grad || grad_hi) && ldg < n))
    return MR_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(logits) % elt_bytes(dtype) ||
      reinterpret_cast<uintptr_t>(grad) % elt_bytes(dtype))
    return MR_ERR_ALIGNMENT;
  const GradOut out{grad, grad_hi, grad_lo};
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    distill_kernel<T><<<unsigned(rows), kDistThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(logits), ld, n, t_logits, t_index, k, temperature, weight, loss, out,
        ldg);
    return launch_status();
  });
}
