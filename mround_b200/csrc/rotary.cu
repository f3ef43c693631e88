// K10 -- rotary positions on query and key heads, forward and transposed.
//
// For the pair of columns (j, j + r/2) (half layout) or (2j, 2j + 1)
// (interleaved) of a head's first r columns, j < r/2, with c and s the token's
// row of the cosine and sine tables:
//   forward     y1 = x1 c - x2 s      y2 = x1 s + x2 c
//   transposed  y1 = x1 c + x2 s      y2 = x2 c - x1 s   (the backward pass)
// in float32, rounded once; columns from r on are copied.  The transposed form
// is the inverse only where c^2 + s^2 = 1: tables may carry a factor (YaRN's
// attention scaling), which the gradient carries too.
//
// HBM-bound: each value is read and written once (16384 tokens x 32 heads of 128
// float32: 92 us, 5.8 TB/s).  A thread keeps one unit of columns (two vectors:
// 16 bytes of each half, or 32 bytes of interleaved pairs), reads its cosines
// and sines once and walks the token's heads four at a time, so that four heads'
// loads are in flight and the tables cost one read per four heads.  A block
// takes as many tokens as fill 128 threads.  A launch takes query and key heads
// together: at one token the launch itself is the cost.
//
// Tensors whose addresses or strides do not divide into 16 bytes, or whose
// halves do not divide into whole vectors, take narrower forms of the same
// kernel: vectors of two columns, or one column at a time.

#include <type_traits>

#include "rowtypes.cuh"

namespace mr {
namespace {

// Two values.
template <typename T>
struct Pair {
  typename std::conditional<sizeof(T) == 4, uint2, uint32_t>::type raw;
  __device__ __forceinline__ void get(float (&f)[2]) const {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(raw.x);
      f[1] = __uint_as_float(raw.y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&raw));
      f[0] = p.x;
      f[1] = p.y;
    } else {
      f[0] = __uint_as_float(raw << 16);
      f[1] = __uint_as_float(raw & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void put(const float (&f)[2]) {
    if constexpr (sizeof(T) == 4) {
      raw = make_uint2(__float_as_uint(f[0]), __float_as_uint(f[1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 p = __floats2half2_rn(f[0], f[1]);
      raw = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[0], f[1]);
      raw = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
};

template <typename T>
struct One {
  T raw;
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f32(raw); }
  __device__ __forceinline__ void put(const float (&f)[1]) { raw = from_f32<T>(f[0]); }
};

template <typename T, int V>
using VecOf = typename std::conditional<
    V == 1, One<T>, typename std::conditional<V == 2, Pair<T>, Vec16<T>>::type>::type;

struct RotaryHeads {
  const void* x;
  void* y;
  int64_t xb, xs, xh;  // strides of batch, position and head, in elements
  int64_t yb, ys, yh;
  int heads;
};

struct RotaryArgs {
  RotaryHeads q, k;
  const float* cosv;
  const float* sinv;
  const void* positions;  // NULL: the index in the sequence
  int64_t table_rows, pos_stride;
  int pos64;
  int64_t tokens;
  int seq, d, r;
};

constexpr int kHeadsAtOnce = 4;

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t b, int s) {
  if (!a.positions) return s;
  const int64_t i = b * a.pos_stride + s;
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[i]
                 : int64_t(static_cast<const int32_t*>(a.positions)[i]);
}

// blockDim.x: column units of a head (rotated units of two vectors first, then
// copied ones of one); blockDim.y: head lanes; blockDim.z: tokens.  V columns
// per vector: 16 bytes, two columns, or one.
template <typename T, bool kInterleaved, bool kTransposed, int V>
__global__ void __launch_bounds__(V * sizeof(T) == 16 ? 256 : V > 1 ? 512 : 1024)
    rotary_kernel(const __grid_constant__ RotaryArgs a) {
  using Vec = VecOf<T, V>;
  using Raw = decltype(Vec::raw);
  const int turned = a.r / (2 * V);  // rotated units per head, V pairs each
  const int u = threadIdx.x;
  const int heads = a.q.heads + a.k.heads;
  const bool rotates = u < turned;
  const int c0 = !rotates ? a.r + (u - turned) * V : kInterleaved ? u * 2 * V : u * V;
  const int c1 = kInterleaved ? c0 + V : c0 + a.r / 2;
  const int64_t step = int64_t(gridDim.x) * blockDim.z;
  for (int64_t t = int64_t(blockIdx.x) * blockDim.z + threadIdx.z; t < a.tokens; t += step) {
    const int64_t b = t / a.seq;
    const int s = int(t - b * a.seq);
    float cs[V], sn[V];
    if (rotates) {
      const int64_t p = position_of(a, b, s);
      if (p >= 0 && p < a.table_rows) {
        const float* cr = a.cosv + p * (a.r / 2) + u * V;
        const float* sr = a.sinv + p * (a.r / 2) + u * V;
        if constexpr (V % 4 == 0) {
#pragma unroll
          for (int i = 0; i < V; i += 4) {
            const float4 c4 = *reinterpret_cast<const float4*>(cr + i);
            const float4 s4 = *reinterpret_cast<const float4*>(sr + i);
            cs[i] = c4.x; cs[i + 1] = c4.y; cs[i + 2] = c4.z; cs[i + 3] = c4.w;
            sn[i] = s4.x; sn[i + 1] = s4.y; sn[i + 2] = s4.z; sn[i + 3] = s4.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            cs[i] = cr[i];
            sn[i] = sr[i];
          }
        }
      } else {  // outside the tables: no angle to turn by
#pragma unroll
        for (int i = 0; i < V; ++i) cs[i] = sn[i] = __int_as_float(0x7fffffff);
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (kTransposed) sn[i] = -sn[i];
    }
    for (int h0 = threadIdx.y; h0 < heads; h0 += blockDim.y * kHeadsAtOnce) {
      const T* src[kHeadsAtOnce];
      T* dst[kHeadsAtOnce];
      Vec v0[kHeadsAtOnce], v1[kHeadsAtOnce];
#pragma unroll
      for (int i = 0; i < kHeadsAtOnce; ++i) {
        int h = h0 + i * blockDim.y;
        src[i] = nullptr;
        if (h >= heads) continue;
        const RotaryHeads& w = h < a.q.heads ? a.q : a.k;
        if (h >= a.q.heads) h -= a.q.heads;
        src[i] = static_cast<const T*>(w.x) + b * w.xb + s * w.xs + h * w.xh;
        dst[i] = static_cast<T*>(w.y) + b * w.yb + s * w.ys + h * w.yh;
        v0[i].raw = *reinterpret_cast<const Raw*>(src[i] + c0);
        if (rotates) v1[i].raw = *reinterpret_cast<const Raw*>(src[i] + c1);
      }
#pragma unroll
      for (int i = 0; i < kHeadsAtOnce; ++i) {
        if (!src[i]) continue;
        if (rotates) {
          float f0[V], f1[V];
          v0[i].get(f0);
          v1[i].get(f1);
          if constexpr (kInterleaved && V > 1) {  // pairs of neighbours in each vector
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float x1 = f0[2 * j], x2 = f0[2 * j + 1];
              f0[2 * j] = x1 * cs[j] - x2 * sn[j];
              f0[2 * j + 1] = x1 * sn[j] + x2 * cs[j];
              const float x3 = f1[2 * j], x4 = f1[2 * j + 1];
              f1[2 * j] = x3 * cs[V / 2 + j] - x4 * sn[V / 2 + j];
              f1[2 * j + 1] = x3 * sn[V / 2 + j] + x4 * cs[V / 2 + j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float x1 = f0[j], x2 = f1[j];
              f0[j] = x1 * cs[j] - x2 * sn[j];
              f1[j] = x1 * sn[j] + x2 * cs[j];
            }
          }
          v0[i].put(f0);
          v1[i].put(f1);
          *reinterpret_cast<Raw*>(dst[i] + c1) = v1[i].raw;
        }
        *reinterpret_cast<Raw*>(dst[i] + c0) = v0[i].raw;
      }
    }
  }
}

// Whether addresses and strides divide into vectors of v columns.
bool heads_divide(const RotaryHeads& h, int v, int elt) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.y);
  return !h.heads || (at % (v * elt) == 0 && h.xb % v == 0 && h.xs % v == 0 && h.xh % v == 0 &&
                      h.yb % v == 0 && h.ys % v == 0 && h.yh % v == 0);
}

template <typename T, bool kInterleaved, bool kTransposed, int V>
int launch_rotary_as(const RotaryArgs& a, cudaStream_t stream) {
  const int heads = a.q.heads + a.k.heads;
  const int units = a.r / (2 * V) + (a.d - a.r) / V;
  int lanes = (heads + kHeadsAtOnce - 1) / kHeadsAtOnce;
  const int most = 256 / units > 0 ? 256 / units : 1;
  if (lanes > most) lanes = most;
  int z = 128 / (units * lanes);  // blockDim.z is at most 64
  z = z < 1 ? 1 : z > 64 ? 64 : z;
  if (z > a.tokens) z = int(a.tokens);
  const int64_t blocks = (a.tokens + z - 1) / z;
  const unsigned grid = unsigned(blocks < 0x7fffffff ? blocks : 0x7fffffff);
  rotary_kernel<T, kInterleaved, kTransposed, V><<<grid, dim3(units, lanes, z), 0, stream>>>(a);
  return launch_status();
}

template <typename T, bool kInterleaved, bool kTransposed>
int launch_rotary(const RotaryArgs& a, cudaStream_t stream) {
  constexpr int kElt = int(sizeof(T)), kWide = 16 / kElt;
  // whole units of two vectors of v columns, and whole vectors of copied ones
  auto divides = [&](int v) {
    return a.r % (2 * v) == 0 && a.d % v == 0 && heads_divide(a.q, v, kElt) &&
           heads_divide(a.k, v, kElt);
  };
  if (divides(kWide) && aligned16(a.cosv) && aligned16(a.sinv))
    return launch_rotary_as<T, kInterleaved, kTransposed, kWide>(a, stream);
  if (divides(2)) return launch_rotary_as<T, kInterleaved, kTransposed, 2>(a, stream);
  return launch_rotary_as<T, kInterleaved, kTransposed, 1>(a, stream);
}

// Operand forms for the decoder block (float32 rows of [q | k | v] heads in,
// bf16 hi/lo head tensors out, and back), for the layouts and head parts that
// the whole-head half-layout kernels of mr_rope_split do not cover.  One block
// walks a token's row; a thread takes V pairs of one head (V = 4 with 16-byte
// accesses, else 1) or, past the rotated columns and in the value heads, 2 V
// columns copied.
__device__ __forceinline__ void split_of(float v, uint16_t& h, uint16_t& l) {
  h = f32_to_bf16(v);
  l = f32_to_bf16(__fsub_rn(v, bf16_to_f32(h)));
}

template <int V>
__device__ __forceinline__ void load_v(const float* p, float (&f)[V]) {
  if constexpr (V == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
  } else {
    f[0] = *p;
  }
}

template <int V>
__device__ __forceinline__ void store_split(uint16_t* hi, uint16_t* lo, int64_t at,
                                            const float (&f)[V]) {
  uint16_t h[V], l[V];
#pragma unroll
  for (int i = 0; i < V; ++i) split_of(f[i], h[i], l[i]);
  if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(hi + at) = make_uint2(uint32_t(h[0]) | (uint32_t(h[1]) << 16),
                                                    uint32_t(h[2]) | (uint32_t(h[3]) << 16));
    *reinterpret_cast<uint2*>(lo + at) = make_uint2(uint32_t(l[0]) | (uint32_t(l[1]) << 16),
                                                    uint32_t(l[2]) | (uint32_t(l[3]) << 16));
  } else {
    hi[at] = h[0];
    lo[at] = l[0];
  }
}

template <int V>
__device__ __forceinline__ void store_v(float* p, const float (&f)[V]) {
  if constexpr (V == 4)
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else
    *p = f[0];
}

struct BlockRotary {
  const float* cosv;
  const float* sinv;
  int S, Hq, Hkv, D, R, interleaved;
  int64_t tokens;
};

// Columns of the unit's two vectors.  Half layout: V columns of each half;
// interleaved: 2 V columns in a row.  Copied units: 2 V columns in a row.
__device__ __forceinline__ void unit_columns(const BlockRotary& a, int u, int V, bool rotated_head,
                                             int* c0, int* c1, int* pair0) {
  const int turned = rotated_head ? a.R / (2 * V) : 0;
  if (u < turned) {
    *pair0 = u * V;
    *c0 = a.interleaved ? u * 2 * V : u * V;
    *c1 = a.interleaved ? *c0 + V : *c0 + a.R / 2;
  } else {
    *pair0 = -1;
    *c0 = (rotated_head ? a.R : 0) + (u - turned) * 2 * V;
    *c1 = *c0 + V;
  }
}

// Rotates V pairs held as two vectors; sgn = 1 forward, -1 transposed.
template <int V>
__device__ __forceinline__ void turn_pairs(const BlockRotary& a, int s, int pair0, float sgn,
                                           float (&x0)[V], float (&x1)[V]) {
  float c[V], sn[V];
  load_v<V>(a.cosv + int64_t(s) * (a.R / 2) + pair0, c);
  load_v<V>(a.sinv + int64_t(s) * (a.R / 2) + pair0, sn);
  if (a.interleaved && V == 4) {  // pairs (0, 1) and (2, 3) of each vector
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float p = x0[2 * j], q = x0[2 * j + 1], r = x1[2 * j], t = x1[2 * j + 1];
      const float sa = sgn * sn[j], sb = sgn * sn[j + V / 2];
      x0[2 * j] = p * c[j] - q * sa;
      x0[2 * j + 1] = p * sa + q * c[j];
      x1[2 * j] = r * c[j + V / 2] - t * sb;
      x1[2 * j + 1] = r * sb + t * c[j + V / 2];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float p = x0[j], q = x1[j], sa = sgn * sn[j];
      x0[j] = p * c[j] - q * sa;
      x1[j] = p * sa + q * c[j];
    }
  }
}

template <int V>
__global__ void __launch_bounds__(256) rotary_split_kernel(
    const float* __restrict__ qkv, const BlockRotary a, uint16_t* __restrict__ q_hi,
    uint16_t* __restrict__ q_lo, uint16_t* __restrict__ k_hi, uint16_t* __restrict__ k_lo,
    uint16_t* __restrict__ v_hi, uint16_t* __restrict__ v_lo) {
  const int per_head = a.D / (2 * V);
  const int H = a.Hq + 2 * a.Hkv;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t b = t / a.S;
    const int s = int(t - b * a.S);
    for (int w = threadIdx.x; w < H * per_head; w += blockDim.x) {
      const int head = w / per_head;
      int c0, c1, pair0;
      unit_columns(a, w - head * per_head, V, head < a.Hq + a.Hkv, &c0, &c1, &pair0);
      const float* src = qkv + (t * H + head) * a.D;
      float x0[V], x1[V];
      load_v<V>(src + c0, x0);
      load_v<V>(src + c1, x1);
      if (pair0 >= 0) turn_pairs<V>(a, s, pair0, 1.f, x0, x1);
      uint16_t *hi, *lo;
      int64_t at;
      if (head < a.Hq) {
        hi = q_hi; lo = q_lo;
        at = ((b * a.Hq + head) * a.S + s) * a.D;
      } else if (head < a.Hq + a.Hkv) {
        hi = k_hi; lo = k_lo;
        at = ((b * a.Hkv + head - a.Hq) * a.S + s) * a.D;
      } else {
        hi = v_hi; lo = v_lo;
        at = ((b * a.Hkv + head - a.Hq - a.Hkv) * a.S + s) * a.D;
      }
      store_split<V>(hi, lo, at + c0, x0);
      store_split<V>(hi, lo, at + c1, x1);
    }
  }
}

template <int V>
__global__ void __launch_bounds__(256) rotary_bwd_split_kernel(
    const float* __restrict__ dq, const float* __restrict__ dk, const float* __restrict__ dv,
    const BlockRotary a, uint16_t* __restrict__ hi, uint16_t* __restrict__ lo,
    float* __restrict__ t32) {
  const int per_head = a.D / (2 * V);
  const int H = a.Hq + 2 * a.Hkv;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t b = t / a.S;
    const int s = int(t - b * a.S);
    for (int w = threadIdx.x; w < H * per_head; w += blockDim.x) {
      const int head = w / per_head;
      int c0, c1, pair0;
      unit_columns(a, w - head * per_head, V, head < a.Hq + a.Hkv, &c0, &c1, &pair0);
      const float* src;
      if (head < a.Hq) src = dq + ((b * a.Hq + head) * a.S + s) * a.D;
      else if (head < a.Hq + a.Hkv) src = dk + ((b * a.Hkv + head - a.Hq) * a.S + s) * a.D;
      else src = dv + ((b * a.Hkv + head - a.Hq - a.Hkv) * a.S + s) * a.D;
      float x0[V], x1[V];
      load_v<V>(src + c0, x0);
      load_v<V>(src + c1, x1);
      if (pair0 >= 0) turn_pairs<V>(a, s, pair0, -1.f, x0, x1);
      const int64_t at = (t * H + head) * a.D;
      if (hi) {
        store_split<V>(hi, lo, at + c0, x0);
        store_split<V>(hi, lo, at + c1, x1);
      }
      if (t32) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x0[i] = tf32_rna(x0[i]);
          x1[i] = tf32_rna(x1[i]);
        }
        store_v<V>(t32 + at + c0, x0);
        store_v<V>(t32 + at + c1, x1);
      }
    }
  }
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

bool block_shape(BlockRotary* a, const float* cosv, const float* sinv, int b, int s, int hq,
                 int hkv, int d, int r, int interleaved) {
  if (!cosv || !sinv || b <= 0 || s <= 0 || hq <= 0 || hkv <= 0 || d <= 0 || d % 2 || r <= 0 ||
      r % 2 || r > d)
    return false;
  *a = BlockRotary{cosv, sinv, s, hq, hkv, d, r, interleaved != 0, int64_t(b) * s};
  return true;
}

// four pairs per thread: the rotated, copied and value columns in eights
bool block_wide(const BlockRotary& a) {
  return a.R % 8 == 0 && a.D % 8 == 0 && aligned16(a.cosv) && aligned16(a.sinv);
}

unsigned token_grid(int64_t tokens) { return unsigned(tokens < 0x7fffffff ? tokens : 0x7fffffff); }

bool take_heads(const mr_rotary_heads* h, RotaryHeads* to) {
  *to = RotaryHeads{};
  if (!h) return true;
  if (!h->x || !h->y || h->heads <= 0) return false;
  to->x = h->x;
  to->y = h->y;
  to->xb = h->x_batch; to->xs = h->x_pos; to->xh = h->x_head;
  to->yb = h->y_batch; to->ys = h->y_pos; to->yh = h->y_head;
  to->heads = h->heads;
  return true;
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" int mr_rotary(const mr_rotary_heads* q, const mr_rotary_heads* k, const float* cosv,
                         const float* sinv, int64_t table_rows, const void* positions,
                         int positions64, int64_t pos_stride, int64_t b, int s, int d, int r,
                         int interleaved, int transposed, int dtype, void* stream) {
  if (!q || !cosv || !sinv || table_rows <= 0 || b <= 0 || s <= 0 || d <= 0 || d > 1024 || r <= 0 ||
      r % 2 || r > d || !known_dtype(dtype))
    return MR_ERR_ARGUMENT;
  RotaryArgs a;
  if (!take_heads(q, &a.q) || !take_heads(k, &a.k)) return MR_ERR_ARGUMENT;
  a.cosv = cosv;
  a.sinv = sinv;
  a.positions = positions;
  a.table_rows = table_rows;
  a.pos_stride = pos_stride;
  a.pos64 = positions64;
  a.tokens = b * s;
  a.seq = s;
  a.d = d;
  a.r = r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (interleaved)
      return transposed ? launch_rotary<T, true, true>(a, st) : launch_rotary<T, true, false>(a, st);
    return transposed ? launch_rotary<T, false, true>(a, st) : launch_rotary<T, false, false>(a, st);
  });
}

extern "C" int mr_rotary_split(const float* qkv, const float* cosv, const float* sinv, int b, int s,
                               int hq, int hkv, int d, int r, int interleaved, uint16_t* q_hi,
                               uint16_t* q_lo, uint16_t* k_hi, uint16_t* k_lo, uint16_t* v_hi,
                               uint16_t* v_lo, void* stream) {
  BlockRotary a;
  if (!qkv || !q_hi || !q_lo || !k_hi || !k_lo || !v_hi || !v_lo ||
      !block_shape(&a, cosv, sinv, b, s, hq, hkv, d, r, interleaved))
    return MR_ERR_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = block_wide(a) && aligned16(qkv) && aligned8(q_hi) && aligned8(q_lo) &&
                    aligned8(k_hi) && aligned8(k_lo) && aligned8(v_hi) && aligned8(v_lo);
  if (wide)
    rotary_split_kernel<4><<<token_grid(a.tokens), 256, 0, st>>>(qkv, a, q_hi, q_lo, k_hi, k_lo,
                                                                 v_hi, v_lo);
  else
    rotary_split_kernel<1><<<token_grid(a.tokens), 256, 0, st>>>(qkv, a, q_hi, q_lo, k_hi, k_lo,
                                                                 v_hi, v_lo);
  return launch_status();
}

extern "C" int mr_rotary_bwd_split(const float* dq, const float* dk, const float* dv,
                                   const float* cosv, const float* sinv, int b, int s, int hq,
                                   int hkv, int d, int r, int interleaved, uint16_t* hi,
                                   uint16_t* lo, float* t32, void* stream) {
  BlockRotary a;
  if (!dq || !dk || !dv || (hi == nullptr) != (lo == nullptr) || (!hi && !t32) ||
      !block_shape(&a, cosv, sinv, b, s, hq, hkv, d, r, interleaved))
    return MR_ERR_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = block_wide(a) && aligned16(dq) && aligned16(dk) && aligned16(dv) &&
                    aligned8(hi) && aligned8(lo) && aligned16(t32);
  if (wide)
    rotary_bwd_split_kernel<4><<<token_grid(a.tokens), 256, 0, st>>>(dq, dk, dv, a, hi, lo, t32);
  else
    rotary_bwd_split_kernel<1><<<token_grid(a.tokens), 256, 0, st>>>(dq, dk, dv, a, hi, lo, t32);
  return launch_status();
}
