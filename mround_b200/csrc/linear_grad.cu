// The element-wise part of K13's backward: dz = dy act'(z) in bf16 or as a bf16
// hi/lo pair (the operand of the two gradient products), and the bias gradient
// sum_t dz.
//
// HBM-bound: z (float32) and dy are read once, dz is written once.  A
// block takes a strip of 256 features and 64 tokens: 64 threads of four
// features by four token lanes.  Bias sums stay in float32 registers, are
// joined in the block and written per strip; a second kernel adds the strips
// in token order, so the result does not depend on timing.  2047 tokens by 11008
// features, tanh GELU, bf16 dy, dz as a pair: 55 us from cold caches, 4.1 TB/s.

#include "rowtypes.cuh"

namespace mr {
namespace {

constexpr int kGradLanes = 4;      // tokens at once per block
constexpr int kGradTokens = 64;    // tokens per strip
constexpr int kGradFeatures = 256; // features per block

// act'(z).  SiLU and the tanh GELU (z times the logistic function of 2u, u' as
// below) take one exponential and one division.
__device__ __forceinline__ float logistic(float v) { return 1.f / (1.f + expf(-v)); }
__device__ __forceinline__ float silu_grad(float z) {
  const float s = logistic(z);
  return s * (1.f + z * (1.f - s));
}
__device__ __forceinline__ float gelu_tanh_grad(float z) {
  const float s = logistic(1.5957691216057308f * (z + 0.044715f * z * z * z));
  // s (1 - s) first: far from zero it is 0 where z^3, or z^2, is infinite
  const float a = z * (s * (1.f - s)) * 1.5957691216057308f;
  return s + (a + a * z * z * 0.134145f);
}
__device__ __forceinline__ float gelu_grad(float z) {
  return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
         z * 0.39894228040143268f * expf(-0.5f * z * z);
}

// d act'(a) for one token's values
template <int V>
__device__ __forceinline__ void times_grad(int act, const float (&d)[V], float (&a)[V]) {
  auto each = [&](auto fn) {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = d[i] * fn(a[i]);
  };
  if (act == MR_ACT_SILU)
    each(silu_grad);
  else if (act == MR_ACT_GELU)
    each(gelu_grad);
  else if (act == MR_ACT_GELU_TANH)
    each(gelu_tanh_grad);
  else
    each([](float) { return 1.f; });
}

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, float (&f)[V]) {
  if constexpr (V == 4 && sizeof(T) == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
  } else if constexpr (V == 4) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(q.x << 16);
    f[1] = __uint_as_float(q.x & 0xFFFF0000u);
    f[2] = __uint_as_float(q.y << 16);
    f[3] = __uint_as_float(q.y & 0xFFFF0000u);
  } else {
    f[0] = to_f32(*p);
  }
}

template <int V>
__device__ __forceinline__ void put_pair(uint16_t* hi, uint16_t* lo, int64_t at,
                                         const float (&f)[V]) {
  uint16_t h[V], l[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = f32_to_bf16(f[i]);
    l[i] = f32_to_bf16(__fsub_rn(f[i], bf16_to_f32(h[i])));
  }
  if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(hi + at) = make_uint2(uint32_t(h[0]) | (uint32_t(h[1]) << 16),
                                                    uint32_t(h[2]) | (uint32_t(h[3]) << 16));
    if (lo)
      *reinterpret_cast<uint2*>(lo + at) = make_uint2(uint32_t(l[0]) | (uint32_t(l[1]) << 16),
                                                    uint32_t(l[2]) | (uint32_t(l[3]) << 16));
  } else {
    hi[at] = h[0];
    if (lo) lo[at] = l[0];
  }
}

// sums: (strips, features of dz) or NULL.  One token at a time and six blocks an
// SM: four tokens' loads in flight per thread cost blocks, and took 1.4 times as
// long.
template <typename T, int V, bool kGated>
__global__ void __launch_bounds__(kGradFeatures, 6) act_grad_kernel(
    const T* __restrict__ dy, int64_t ldy, const float* __restrict__ z, int64_t ldz,
    int64_t toks, int feats, int act, uint16_t* __restrict__ hi, uint16_t* __restrict__ lo,
    int64_t ldo, float* __restrict__ sums) {
  constexpr int kOut = kGated ? 2 : 1;
  constexpr int kUnits = kGradFeatures / 4;
  __shared__ float part[kGradLanes][kOut][kUnits * V];
  const int u = threadIdx.x % kUnits, row = threadIdx.x / kUnits;
  const int f = (blockIdx.x * kUnits + u) * V;
  const int64_t t0 = int64_t(blockIdx.y) * kGradTokens;
  const int64_t t1 = t0 + kGradTokens < toks ? t0 + kGradTokens : toks;
  float acc[kOut][V] = {};  // z NULL: no activation
  if (f < feats) {
    for (int64_t t = t0 + row; t < t1; t += kGradLanes) {
      float d[V], a[V], b[V];
      load_row<T, V>(dy + t * ldy + f, d);
      if (z) load_row<float, V>(z + t * ldz + f, a);
      if constexpr (kGated) {
        load_row<float, V>(z + t * ldz + feats + f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = logistic(a[i]);
          const float gate = d[i] * b[i] * (s * (1.f + a[i] * (1.f - s)));
          b[i] = d[i] * (a[i] * s);
          a[i] = gate;
          acc[1][i] += b[i];
        }
        if (hi) put_pair<V>(hi, lo, t * ldo + feats + f, b);
      } else if (z) {
        times_grad(act, d, a);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = d[i];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[0][i] += a[i];
      if (hi) put_pair<V>(hi, lo, t * ldo + f, a);
    }
  }
  if (!sums) return;
#pragma unroll
  for (int o = 0; o < kOut; ++o)
#pragma unroll
    for (int i = 0; i < V; ++i) part[row][o][u * V + i] = acc[o][i];
  __syncthreads();
  if (row == 0 && f < feats) {
#pragma unroll
    for (int o = 0; o < kOut; ++o)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kGradLanes; ++r) s += part[r][o][u * V + i];
        sums[int64_t(blockIdx.y) * feats * kOut + o * feats + f + i] = s;
      }
  }
}

__global__ void __launch_bounds__(256) add_strips_kernel(const float* __restrict__ sums, int strips,
                                                         int n, float* __restrict__ out) {
  const int f = blockIdx.x * 256 + threadIdx.x;
  if (f >= n) return;
  float s = 0.f;
  for (int i = 0; i < strips; ++i) s += sums[int64_t(i) * n + f];
  out[f] = s;
}

int64_t strips_of(int64_t toks) { return (toks + kGradTokens - 1) / kGradTokens; }

template <typename T, int V>
int launch_act_grad(const void* dy, int64_t ldy, const float* z, int64_t ldz, int64_t toks,
                    int feats, int act, uint16_t* hi, uint16_t* lo, int64_t ldo, float* sums,
                    cudaStream_t stream) {
  const int units = (feats + V - 1) / V;
  const dim3 grid((units + kGradFeatures / 4 - 1) / (kGradFeatures / 4), unsigned(strips_of(toks)));
  const T* d = static_cast<const T*>(dy);
  if (act == MR_ACT_SWIGLU)
    act_grad_kernel<T, V, true><<<grid, kGradFeatures, 0, stream>>>(d, ldy, z, ldz, toks, feats, act,
                                                                    hi, lo, ldo, sums);
  else
    act_grad_kernel<T, V, false><<<grid, kGradFeatures, 0, stream>>>(d, ldy, z, ldz, toks, feats,
                                                                     act, hi, lo, ldo, sums);
  return launch_status();
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" size_t mr_act_grad_workspace_bytes(int64_t toks, int64_t feats, int act) {
  if (toks <= kGradTokens || feats <= 0) return 0;  // one strip is the sum itself
  return size_t(strips_of(toks)) * size_t(feats) * (act == MR_ACT_SWIGLU ? 2 : 1) * sizeof(float);
}

extern "C" int mr_act_grad(const void* dy, int dy_dtype, int64_t ldy, const float* z, int64_t ldz,
                           int64_t toks, int64_t feats, int act, uint16_t* hi, uint16_t* lo,
                           int64_t ldo, float* bias_grad, void* workspace, void* stream) {
  const int rows = act == MR_ACT_SWIGLU ? 2 : 1;
  if (!dy || (!z && act != MR_ACT_NONE) || (!hi && (lo || !bias_grad)) || toks <= 0 ||
      feats <= 0 || feats > 0x3fffffff || act < MR_ACT_NONE || act > MR_ACT_SWIGLU ||
      ldy < feats || (z && ldz < rows * feats) ||
      (hi && ldo < rows * feats) || (dy_dtype != MR_F32 && dy_dtype != MR_BF16) ||
      strips_of(toks) > 65535)
    return MR_ERR_ARGUMENT;
  const bool one_strip = toks <= kGradTokens;
  if (bias_grad && !workspace && !one_strip) return MR_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* sums = !bias_grad ? nullptr : one_strip ? bias_grad : static_cast<float*>(workspace);
  const bool wide = feats % 4 == 0 && ldy % 4 == 0 && (!z || ldz % 4 == 0) && (!hi || ldo % 4 == 0) &&
                    aligned16(z) &&
                    ((reinterpret_cast<uintptr_t>(hi) | reinterpret_cast<uintptr_t>(lo)) & 7u) == 0 &&
                    (reinterpret_cast<uintptr_t>(dy) & (dy_dtype == MR_F32 ? 15u : 7u)) == 0;
  int status;
  const int n = int(feats);
  if (dy_dtype == MR_F32)
    status = wide ? launch_act_grad<float, 4>(dy, ldy, z, ldz, toks, n, act, hi, lo, ldo, sums, st)
                  : launch_act_grad<float, 1>(dy, ldy, z, ldz, toks, n, act, hi, lo, ldo, sums, st);
  else
    status = wide ? launch_act_grad<__nv_bfloat16, 4>(dy, ldy, z, ldz, toks, n, act, hi, lo, ldo,
                                                      sums, st)
                  : launch_act_grad<__nv_bfloat16, 1>(dy, ldy, z, ldz, toks, n, act, hi, lo, ldo,
                                                      sums, st);
  if (status != MR_OK || !bias_grad || one_strip) return status;
  add_strips_kernel<<<unsigned((rows * feats + 255) / 256), 256, 0, st>>>(
      sums, int(strips_of(toks)), int(rows * feats), bias_grad);
  return launch_status();
}
