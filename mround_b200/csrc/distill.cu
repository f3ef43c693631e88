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
// HBM-bound: the logits are read once and the gradient is written once.  A CTA
// takes a row: an online maximum and sum of exponentials, per thread, the next
// loads in flight while one step is summed; for the gradient it leaves the
// first part of the row in its shared memory, each thread its own vectors, and
// reads the rest again while it is in L2 (loads of the first pass may stay
// there, the last ones and the gradient's stores go first).  Reading whole rows
// twice, two CTAs per SM with rows of 608 KB, exceeded L2: 592 us for 2047 x
// 152064 float32, three transfers per value; now 482 us, 5.2 TB/s of the
// two.  One warp computes the teacher's side meanwhile.  Few rows are divided
// among the CTAs of a cluster, which join (max, sum) over distributed shared
// memory.
//
// Exponentials are 2^(c x - a), c = log2(e) / T, a = round(c max): one fused
// rounding of the exponent, and every term uses the same a, so its rounding
// cancels in q.  It has to be small for that: below |c max| = 2^24 the largest
// term is 2^+-0.5, but at 2^31 it would be 2^+-64, and further out infinite or
// nothing.  So a running maximum starts at -2^24 / c, below which a value adds
// to the sum without becoming the maximum, and a row whose maximum is not
// between these bounds (a row masked whole, say) is summed again as
// 2^((x - max) c).
// Sums are float32 per thread and joined in float64 in a fixed order; the K
// terms, and the logarithms, are in float64, because the loss is a difference
// of logarithms of size ~10.  The kept columns are corrected after the row is
// written, each by one thread, duplicates summed, so nothing depends on an
// order of atomics.

#include <type_traits>

#include "rowtypes.cuh"
#include "sm100.cuh"

namespace mr {
namespace {

constexpr int kDistUnroll = 4;
constexpr int kDistMaxK = 256;
constexpr float kFarExponent = 16777216.f;  // largest |c max| of the fused form

struct DistShared {
  float m[32];           // per streaming warp
  double s[32];
  float part_m[3];       // this CTA's, by round
  double part_s[3];
  float all_m;
  double all_s;
  double p[kDistMaxK], log_p[kDistMaxK];
  float x[kDistMaxK];
  int64_t col[kDistMaxK];
  int bad, empty;
};

// 2^v (within 2^-22; results below 2^-126 are 0)
__device__ __forceinline__ float pow2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float warp_top(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// (max, sum of exponentials relative to it) of one thread's values.  The
// maximum starts at `lowest`, whose exponent is small enough for the fused form.
struct Online {
  float m, s = 0.f;
  __device__ __forceinline__ explicit Online(float lowest) : m(lowest) {}
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], float c) {
    float top = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
    if (top > m) {
      s *= pow2(__fmul_rn(m, c) - __fmul_rn(top, c));
      m = top;
    }
    const float a = __fmul_rn(m, c);
    float part[4] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) part[i & 3] += pow2(__fmaf_rn(f[i], c, -a));
    s += (part[0] + part[1]) + (part[2] + part[3]);
  }
};

// (max, sum relative to round(c max)) of a warp's lanes, to every lane.
__device__ __forceinline__ void warp_join(float c, float* m, double* s) {
  const float top = warp_top(*m);
  *s = warp_add(*s * double(pow2(__fmul_rn(*m, c) - __fmul_rn(top, c))));
  *m = top;
}

// Joins every streaming thread's (m, s) over the CTA and the cluster, in a
// fixed order.  Each round has slots of its own.  All threads of the cluster
// call it; |m c| is at most kFarExponent unless the sum is to be formed again.
template <int kWarps>
__device__ void join(DistShared& sh, int round, int parts, bool streams, float m, float s, float c,
                     float* top, double* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sd = double(s);
  if (streams) {
    warp_join(c, &m, &sd);
    if (lane == 0) {
      sh.m[warp] = m;
      sh.s[warp] = sd;
    }
  }
  __syncthreads();
  if (warp == 0) {
    m = sh.m[lane < kWarps ? lane : 0];
    sd = lane < kWarps ? sh.s[lane] : 0.0;
    warp_join(c, &m, &sd);
    if (lane == 0) {
      sh.part_m[round] = m;
      sh.part_s[round] = sd;
    }
    __syncwarp();
  }
  if (parts > 1) {
    __syncwarp();
    cluster_sync_all();
    if (warp == 0) {
      const int from = lane < parts ? lane : 0;
      m = ld_cluster(map_rank(smem_u32(&sh.part_m[round]), from));
      sd = ld_cluster_f64(map_rank(smem_u32(&sh.part_s[round]), from));
      if (lane >= parts) sd = 0.0;
      warp_join(c, &m, &sd);
      if (lane == 0) {
        sh.all_m = m;
        sh.all_s = sd;
      }
    }
    __syncthreads();
    *top = sh.all_m;
    *total = sh.all_s;
  } else {
    __syncthreads();
    *top = sh.part_m[round];
    *total = sh.part_s[round];
  }
  // the joined values are read before a later round writes them: its first
  // barrier follows
}

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
    __stcs(reinterpret_cast<uint4*>(static_cast<T*>(o.grad) + at), v.raw);
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
      __stcs(reinterpret_cast<uint2*>(o.hi + at) + i, make_uint2(h[2 * i], h[2 * i + 1]));
      __stcs(reinterpret_cast<uint2*>(o.lo + at) + i, make_uint2(l[2 * i], l[2 * i + 1]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) put_one<T>(o, at + i, g[i]);
  }
}

// The teacher's side of a row, by one warp: p, log p, the student's logits at
// the kept columns.
template <typename T>
__device__ void teacher(DistShared& sh, const T* row, int n, const float* t_logits,
                        const int64_t* t_index, int k, double inv_temperature, float c) {
  const int lane = threadIdx.x & 31;
  constexpr int kEach = kDistMaxK / 32;
  float t[kEach];
  float top = -INFINITY;
  bool bad = false, nan = false;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = i * 32 + lane;
    t[i] = -INFINITY;
    if (j < k) {
      const int64_t col = t_index[j];
      sh.col[j] = col;
      bad |= col >= n;
      if (col >= 0 && col < n) {
        t[i] = t_logits[j];
        sh.x[j] = to_f32(row[col]);
        nan |= t[i] != t[i];
      }
    }
    top = fmaxf(top, t[i]);
  }
  top = warp_top(top);
  // p to float32's own precision: an error of p moves the loss by that error
  // of each term; log p, which does not cancel that way, in float64
  float p[kEach];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    p[i] = t[i] == -INFINITY ? 0.f : pow2((t[i] - top) * c);
    sum += double(p[i]);
  }
  sum = warp_add(sum);
  const double log_sum = log(sum), inv = 1.0 / sum;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = i * 32 + lane;
    if (j < k) {
      sh.p[j] = double(p[i]) * inv;
      sh.log_p[j] = (double(t[i]) - double(top)) * inv_temperature - log_sum;
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) {
    sh.bad = bad;
    sh.empty = top == -INFINITY && !nan && !bad;
  }
}

struct DistArgs {
  const void* logits;  // may be the gradient's own storage
  int64_t ld;
  int n, k, parts, keep;  // keep: vectors of the share that stay in shared memory
  const float* t_logits;
  const int64_t* t_index;
  double temperature, inv_temperature;
  float c;    // log2(e) / T
  float far;  // kFarExponent / c
  const float* weight;
  float* loss;
  GradOut out;
  int64_t ldg;
};

// THREADS streaming threads and the teacher's warp.
template <typename T, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS + 32, CTAS)
    distill_kernel(const __grid_constant__ DistArgs g) {
  __shared__ DistShared sh;
  extern __shared__ uint4 stash[];
  constexpr int kN = Vec16<T>::kN;
  constexpr int kStep = THREADS * kDistUnroll;
  static_assert(THREADS % 32 == 0 && THREADS + 32 <= 1024, "whole warps, the teacher's apart");
  const int tid = threadIdx.x;
  const bool streams = tid < THREADS;
  const int rank = g.parts > 1 ? int(cluster_rank()) : 0;
  const int64_t r = blockIdx.x / g.parts;
  const T* row = static_cast<const T*>(g.logits) + r * g.ld;
  const bool want_grad = g.out.grad || g.out.hi;
  const RowSpan<T> span(row, g.n);
  // this CTA's vectors; rank 0 takes the columns outside the vectors too
  const int v0 = int(int64_t(span.vecs) * rank / g.parts);
  const int v1 = int(int64_t(span.vecs) * (rank + 1) / g.parts);
  const int loose = rank == 0 ? span.loose : 0;
  // stores as wide as the loads where the gradient's row lies as the logits' does
  const int64_t g0 = r * g.ldg;
  bool wide;
  if (g.out.grad)
    wide = (reinterpret_cast<uintptr_t>(static_cast<T*>(g.out.grad) + g0 + span.head) & 15u) == 0;
  else
    wide = ((reinterpret_cast<uintptr_t>(g.out.hi + g0 + span.head) |
             reinterpret_cast<uintptr_t>(g.out.lo + g0 + span.head)) & 7u) == 0;
  const float w = g.weight ? g.weight[r] : 1.f;
  const float c = g.c;
  bool zeros = w == 0.f;  // the same in the whole cluster
  float top = 0.f;
  double total = 1.0;
  bool far = false;
  if (!zeros) {
    Online on(-g.far);
    if (!streams) {
      teacher(sh, row, g.n, g.t_logits + r * g.k, g.t_index + r * g.k, g.k,
              g.inv_temperature, c);
    } else {
      if (tid < loose) {
        const float f[1] = {to_f32(row[span.loose_col(tid)])};
        on.add(f, c);
      }
      // whole steps, the next one's loads in flight while one is summed
      const int steps = (v1 - v0) / kStep;
      int i = v0 + tid;
      auto load = [&](Vec16<T>(&v)[kDistUnroll], int at) {
        if (want_grad) {
#pragma unroll
          for (int u = 0; u < kDistUnroll; ++u) v[u].raw = __ldcg(span.body + at + u * THREADS);
        } else {
#pragma unroll
          for (int u = 0; u < kDistUnroll; ++u) v[u].raw = __ldcs(span.body + at + u * THREADS);
        }
      };
      auto take = [&](const Vec16<T>(&v)[kDistUnroll], int at) {
        if (at - v0 < g.keep) {  // whole steps are kept
#pragma unroll
          for (int u = 0; u < kDistUnroll; ++u) stash[at + u * THREADS - v0] = v[u].raw;
        }
#pragma unroll
        for (int u = 0; u < kDistUnroll; u += 2) {
          float f0[kN], f1[kN], f[2 * kN];
          v[u].get(f0);
          v[u + 1].get(f1);
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            f[j] = f0[j];
            f[kN + j] = f1[j];
          }
          on.add(f, c);
        }
      };
      Vec16<T> even[kDistUnroll], odd[kDistUnroll];
      if (steps > 0) load(even, i);
      for (int n = 0; n < steps; n += 2, i += 2 * kStep) {
        if (n + 1 < steps) load(odd, i + kStep);
        take(even, i);
        if (n + 1 == steps) {
          i += kStep;
          break;
        }
        if (n + 2 < steps) load(even, i + 2 * kStep);
        take(odd, i + kStep);
      }
      for (; i < v1; i += THREADS) {
        Vec16<T> v;
        v.raw = __ldcg(span.body + i);
        if (i - v0 < g.keep) stash[i - v0] = v.raw;
        float f[kN];
        v.get(f);
        on.add(f, c);
      }
    }
    join<THREADS / 32>(sh, 0, g.parts, streams, on.m, on.s, c, &top, &total);
    zeros = sh.empty;
    far = !(top > -g.far && top < g.far);
    if (far) {  // the maximum alone, then the sum relative to it
      float m = -INFINITY, s = 0.f;
      if (streams) {
        if (tid < loose) m = to_f32(row[span.loose_col(tid)]);
        for (int i = v0 + tid; i < v1; i += THREADS) {
          Vec16<T> v;
          v.raw = span.body[i];
          float f[kN];
          v.get(f);
#pragma unroll
          for (int j = 0; j < kN; ++j) m = fmaxf(m, f[j]);
        }
      }
      double no_sum;
      float no_top;
      join<THREADS / 32>(sh, 1, g.parts, streams, m, 0.f, 0.f, &top, &no_sum);
      if (streams) {
        if (tid < loose) s = pow2((to_f32(row[span.loose_col(tid)]) - top) * c);
        for (int i = v0 + tid; i < v1; i += THREADS) {
          Vec16<T> v;
          v.raw = span.body[i];
          float f[kN];
          v.get(f);
#pragma unroll
          for (int j = 0; j < kN; ++j) s += pow2((f[j] - top) * c);
        }
      }
      join<THREADS / 32>(sh, 2, g.parts, streams, 0.f, s, 0.f, &no_top, &total);
    }
  }
  const float a = far ? 0.f : __fmul_rn(top, c);
  auto power = [&](float x) { return far ? pow2((x - top) * c) : pow2(__fmaf_rn(x, c, -a)); };
  const float nan = __int_as_float(0x7fffffff);
  const bool bad = !zeros && sh.bad;
  if (g.loss && rank == 0 && !streams) {
    double term = 0.0;
    if (!zeros) {
      const double log_total = log2(total);
      for (int j = tid - THREADS; j < g.k; j += 32) {
        const double p = sh.p[j];
        if (p > 0.0) {
          const double e = far ? (double(sh.x[j]) - double(top)) * double(c)
                               : double(sh.x[j]) * double(c) - double(a);
          term += p * (sh.log_p[j] - 0.69314718055994530942 * (e - log_total));
        } else if (p != p) {
          term = p;
        }
      }
      term = warp_add(term);
    }
    if (tid == THREADS)
      g.loss[r] = bad ? nan : float(double(w) * g.temperature * g.temperature * term);
  }
  if (want_grad) {
    const float scale = bad ? nan : float(double(w) * g.temperature);
    const float norm = float(double(scale) / total);
    if (streams && zeros) {
      const float f[kN] = {};
      for (int i = v0 + tid; i < v1; i += THREADS)
        put_vec<T>(g.out, g0 + span.head + int64_t(i) * kN, wide, f);
      if (tid < loose) put_one<T>(g.out, g0 + span.loose_col(tid), 0.f);
    } else if (streams) {
      auto write = [&](auto pw) {
        auto one = [&](int i, Vec16<T> v) {
          float f[kN];
          v.get(f);
#pragma unroll
          for (int j = 0; j < kN; ++j) f[j] = pw(f[j]) * norm;
          put_vec<T>(g.out, g0 + span.head + int64_t(i) * kN, wide, f);
        };
        const int kept = min(v0 + g.keep, v1);
        for (int i = kept + tid; i < v1; i += kStep) {  // from L2, for the last time
          Vec16<T> v[kDistUnroll];
#pragma unroll
          for (int u = 0; u < kDistUnroll; ++u)
            if (i + u * THREADS < v1) v[u].raw = __ldcs(span.body + i + u * THREADS);
#pragma unroll
          for (int u = 0; u < kDistUnroll; ++u)
            if (i + u * THREADS < v1) one(i + u * THREADS, v[u]);
        }
#pragma unroll 4
        for (int i = v0 + tid; i < kept; i += THREADS) {
          Vec16<T> v;
          v.raw = stash[i - v0];
          one(i, v);
        }
      };
      if (far)
        write([&](float x) { return pow2((x - top) * c); });
      else
        write([&](float x) { return pow2(__fmaf_rn(x, c, -a)); });
      if (tid < loose) {
        const int col = span.loose_col(tid);
        put_one<T>(g.out, g0 + col, power(to_f32(row[col])) * norm);
      }
    }
    if (!zeros) {
      __syncthreads();  // the kept columns' corrections follow the row
      for (int j = tid; j < g.k; j += THREADS + 32) {
        const int64_t col = sh.col[j];
        if (col < 0 || col >= g.n) continue;
        const int64_t at = col - span.head;
        const bool in_vecs = at >= 0 && at < int64_t(span.vecs) * kN;
        if (in_vecs ? at / kN < v0 || at / kN >= v1 : rank != 0) continue;  // another CTA's
        double mass = 0.0;
        bool first = true;
        for (int i = 0; i < g.k; ++i) {
          if (sh.col[i] != col) continue;
          if (i < j) first = false;
          mass += sh.p[i];
        }
        if (first) {
          const double q = double(power(sh.x[j])) / total;
          put_one<T>(g.out, g0 + col, float((q - mass) * double(scale)));
        }
      }
    }
  }
  // no CTA leaves while another may still read its (max, sum)
  if (g.parts > 1) {
    __syncwarp();
    cluster_sync_all();
  }
}

// CTAs per row.  One is best as long as the rows fill the device: a cluster's
// barriers and joint scheduling cost a CTA about 9 us (2047 x 152064 float32
// with whole shares kept: 8 CTAs per row 823 us, one CTA 482 us).  Fewer rows
// than half of the SMs are divided, down to shares of 8 KB; long rows up to
// two CTAs per SM (74 x 152064 float32, loss: 20.5 us with 2, 30.8 with 1).
int parts_of(int64_t rows, int64_t row_bytes) {
  int parts = 1;
  while (parts < 8 && row_bytes / (parts * 2) >= 8192 &&
         (rows * parts * 2 <= sm_count() ||
          (rows * parts * 2 <= 2 * sm_count() && row_bytes / (parts * 2) >= 128 * 1024)))
    parts *= 2;
  return parts;
}

// keep_bytes: shared memory for the part of the gradient's row that is not
// read again.
template <typename T, int THREADS, int CTAS>
int launch_distill(DistArgs g, int64_t rows, int64_t keep_bytes, cudaStream_t stream) {
  const int64_t row_bytes = int64_t(g.n) * int64_t(sizeof(T));
  g.parts = parts_of(rows, row_bytes);
  if (rows * g.parts > 0x7fffffff) return MR_ERR_ARGUMENT;
  // whole steps of THREADS * kDistUnroll vectors, no more than the share
  constexpr int64_t kStep = THREADS * kDistUnroll;
  g.keep = 0;
  if (g.out.grad || g.out.hi) {
    const int64_t share = (row_bytes / 16 / g.parts + 1 + kStep - 1) / kStep;
    const int64_t most = keep_bytes / (kStep * 16);
    g.keep = int((share < most ? share : most) * kStep);
  }
  static std::atomic<bool> configured[kMaxDevices];
  auto kernel = distill_kernel<T, THREADS, CTAS>;
  const int status = raise_smem(kernel, 217 * 1024, configured);
  if (status != MR_OK) return status;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * g.parts));
  cfg.blockDim = dim3(THREADS + 32);
  cfg.dynamicSmemBytes = size_t(g.keep) * 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(g.parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, g);
  if (err != cudaSuccess) {
    set_cuda_error(err);
    cudaGetLastError();
    return MR_ERR_LAUNCH;
  }
  return launch_status();
}

}  // namespace
}  // namespace mr

using namespace mr;

extern "C" int mr_distill_topk(const void* logits, int64_t rows, int n, int64_t ld, int dtype,
                               const float* t_logits, const int64_t* t_index, int k,
                               double temperature, const float* weight, float* loss, void* grad,
                               uint16_t* grad_hi, uint16_t* grad_lo, int64_t ldg, void* stream) {
  if (!logits || !t_logits || !t_index || rows <= 0 || rows > 0x7fffffff || n <= 0 || ld < n ||
      k <= 0 || k > kDistMaxK || !known_dtype(dtype) || !(temperature >= 1e-3) ||
      !(temperature <= 1e3))
    return MR_ERR_ARGUMENT;
  if ((grad_hi == nullptr) != (grad_lo == nullptr) || (grad && grad_hi) ||
      (!loss && !grad && !grad_hi) || ((grad || grad_hi) && ldg < n))
    return MR_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(logits) % elt_bytes(dtype) ||
      reinterpret_cast<uintptr_t>(grad) % elt_bytes(dtype))
    return MR_ERR_ALIGNMENT;
  DistArgs g;
  g.logits = logits;
  g.ld = ld;
  g.n = n;
  g.k = k;
  g.t_logits = t_logits;
  g.t_index = t_index;
  g.temperature = temperature;
  g.inv_temperature = 1.0 / temperature;
  g.c = float(1.4426950408889634 / temperature);
  g.far = kFarExponent / g.c;
  g.weight = weight;
  g.loss = loss;
  g.out = GradOut{grad, grad_hi, grad_lo};
  g.ldg = ldg;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int64_t row_bytes = int64_t(n) * int64_t(sizeof(T));
    // Block size, measured: rows of up to 16 KB, small blocks and many rows
    // per SM.  The loss alone, 224 + 32 threads four to an SM (511 x 50257
    // float32 28 us, 480 + 32 two to an SM 31).  The gradient of rows of up to
    // 400 KB, 480 + 32 threads two to an SM (2047 x 152064 bf16 266 us; 736 +
    // 32 one to an SM 281); longer rows one to an SM, whose rows in flight fit
    // L2 beside the 200 KB each keeps (float32 482 us; two to an SM 566).
    if (row_bytes <= 16384) return launch_distill<T, 96, 8>(g, rows, 16384, st);
    if (!grad && !grad_hi) return launch_distill<T, 224, 4>(g, rows, 0, st);
    if (row_bytes <= 400 * 1024) return launch_distill<T, 480, 2>(g, rows, 92 * 1024, st);
    return launch_distill<T, 736, 1>(g, rows, 200 * 1024, st);
  });
}
