// K11 -- the k largest values of each row, with their columns.
//
// Order: larger value first, NaN above everything, equal values (and +0 / -0)
// by lowest column.  HBM-bound: a row is read once, the next step's loads in
// flight while one is looked over.
//
// A CTA streams its row with 16-byte loads and keeps a lower bound F of the
// k-th largest value: each thread keeps the two largest of its steps' maxima,
// each of the W warps finds the ceil(k / W)-th largest of its 64, and F is the
// smallest of these -- at least k values are >= F, so what is below F cannot be
// among the k largest.  A step (four vectors a lane) whose maximum reaches F in
// any lane of the warp is compared with F whole, two values an instruction, into
// one mask per lane; values not below F go to the warp's list in shared memory,
// one of each lane's at a time.  (1024 x 152064 bf16: each thread appending its
// own, unrolled, kept the warps waiting for instructions, 133 us; vector by
// vector 82; now 59 us, 5.3 TB/s of the 6.5 a copy reaches.)  F is
// refreshed when the part read has doubled, so a row in no special order lists
// little more than k values per doubling.  At the end the list is cut to the
// last F, and each survivor's rank is the number of listed keys above it
// (value, then column: all keys differ), which is also its place in the
// output: no sort.
//
// Few rows are divided among the CTAs of a cluster: the largest of their F is
// a bound for the whole row, and each ranks its survivors among everyone's.
//
// Of values equal to F a warp lists the first k only, counting them where they
// come in numbers, so that a constant or fully masked row costs little more than
// another.  A row whose list overflows all the same (a rising row) takes the
// exact way instead: four 8-bit radix passes over the row (from L2) find the k-th
// key and the number above it; the values above it, and the first columns equal
// to it, form the list.
//
// Results do not depend on the order in which threads append to the list.

#include <cuda_fp16.h>

#include <type_traits>

#include "rowtypes.cuh"
#include "sm100.cuh"

namespace mr {
namespace {

constexpr int kTopUnroll = 4;     // 16-byte loads per thread and step
constexpr int kTopWarpList = 512; // values a warp lists while streaming
constexpr int kTopShort = 1664;   // of them, not below the last F
constexpr int kTopMaxK = 256;
constexpr uint32_t kKeyLowest = 0x007FFFFFu;  // of -inf; empty slots are below

template <int kWarps>
struct TopShared {
  static constexpr int kList = kWarps * kTopWarpList;
  unsigned long long list[kList];  // per warp; then everyone's survivors
  unsigned long long cut[kTopShort];
  unsigned int hist[256];
  unsigned int part[8];
  int warp_sum[8];
  int listed[8], kept;
  unsigned int floor_key, digit, above;  // floor_key: read by the cluster
  int over;
};

// Order-preserving 32-bit key; NaN is the largest, -0 equals +0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 + 0 is +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __int_as_float(0x7fffffff);
  if (key <= kKeyLowest) return -INFINITY;
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ unsigned long long full_key(float v, int col) {
  return (static_cast<unsigned long long>(key_of(v)) << 32) | uint32_t(0x7FFFFFFF - col);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest value of a vector, NaN if it holds one.
template <typename T>
__device__ __forceinline__ float vec_max(const Vec16<T>& v) {
  if constexpr (sizeof(T) == 4) {
    float f[4];
    v.get(f);
    return max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3]));
  } else if constexpr (std::is_same<T, __half>::value) {
    const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
    const __half2* h = reinterpret_cast<const __half2*>(w);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    const float2 f = __half22float2(m);
    return max_nan(f.x, f.y);
  } else {
    const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
}

// The larger value in each half, NaN if either is.
template <typename T>
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
  using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const P m = __hmax2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// The largest value of a step's vectors, NaN if they hold one.
template <typename T>
__device__ __forceinline__ float step_max(const Vec16<T> (&v)[kTopUnroll]) {
  if constexpr (sizeof(T) == 4) {
    float top = vec_max<T>(v[0]);
#pragma unroll
    for (int u = 1; u < kTopUnroll; ++u) top = max_nan(top, vec_max<T>(v[u]));
    return top;
  } else {  // pairs as long as there are several
    Vec16<T> m = v[0];
#pragma unroll
    for (int u = 1; u < kTopUnroll; ++u) {
      m.raw.x = pair_max<T>(m.raw.x, v[u].raw.x);
      m.raw.y = pair_max<T>(m.raw.y, v[u].raw.y);
      m.raw.z = pair_max<T>(m.raw.z, v[u].raw.z);
      m.raw.w = pair_max<T>(m.raw.w, v[u].raw.w);
    }
    return vec_max<T>(m);
  }
}

// Bit b: the value of word b & 15 of a step's vectors (its upper half for
// b >= 16, of 2-byte types) is not below bar.
template <typename T>
__device__ __forceinline__ uint32_t not_below(const Vec16<T> (&v)[kTopUnroll], float bar) {
  static_assert(kTopUnroll == 4, "16 words a step");
  uint32_t below = 0;
  auto each = [&](auto one) {
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      below |= one(v[u].raw.x) << (4 * u) | one(v[u].raw.y) << (4 * u + 1) |
               one(v[u].raw.z) << (4 * u + 2) | one(v[u].raw.w) << (4 * u + 3);
    }
  };
  if constexpr (sizeof(T) == 4) {
    each([&](uint32_t w) { return __uint_as_float(w) < bar ? 1u : 0u; });
    return ~below & 0xFFFFu;
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 b = __half2half2(__float2half_ru(bar));  // the first value not below
    each([&](uint32_t w) {
      return __hlt2_mask(*reinterpret_cast<const __half2*>(&w), b) & 0x00010001u;
    });
    return ~below;
  } else {
    const __nv_bfloat162 b = __bfloat162bfloat162(__float2bfloat16_ru(bar));
    each([&](uint32_t w) {
      return __hlt2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), b) & 0x00010001u;
    });
    return ~below;
  }
}

// The value of bit b, and its column from the step's first one of this lane
// (vectors `stride` columns apart).
template <typename T>
__device__ __forceinline__ float value_at(const Vec16<T> (&v)[kTopUnroll], int b, int stride,
                                          int* col) {
  const int u = b >> 2 & 3, q = b & 3;
  const uint4 r = u < 2 ? (u == 0 ? v[0].raw : v[1].raw) : (u == 2 ? v[2].raw : v[3].raw);
  const uint32_t w = q < 2 ? (q == 0 ? r.x : r.y) : (q == 2 ? r.z : r.w);
  if constexpr (sizeof(T) == 4) {
    *col = u * stride + q;
    return __uint_as_float(w);
  } else {
    *col = u * stride + 2 * q + (b >> 4);
    const uint16_t h = uint16_t(b & 16 ? w >> 16 : w);
    if constexpr (std::is_same<T, __half>::value)
      return __half2float(__ushort_as_half(h));
    else
      return bf16_to_f32(h);
  }
}

// The smallest, over the warps, of the each-th largest of the lanes' two keys
// (first >= second; 0 where a lane has none); to every thread.
template <int kWarps>
__device__ __forceinline__ uint32_t floor_of(uint32_t first, uint32_t second, int each,
                                             unsigned int* part) {
  const int lane = threadIdx.x & 31;
  uint32_t top = 0;
#pragma unroll 1
  for (int i = 0; i < each; ++i) {
    top = __reduce_max_sync(0xffffffffu, first);
    const unsigned int who = __ballot_sync(0xffffffffu, first == top);
    if (lane == __ffs(who) - 1) {
      first = second;
      second = 0;
    }
  }
  __syncthreads();  // the last reader of part is done
  if (lane == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  uint32_t all = part[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) all = min(all, part[i]);
  return all;
}

// A vector of -inf, in the place of one past the row.
template <typename T>
__device__ __forceinline__ uint4 lowest_vec() {
  const uint32_t w = sizeof(T) == 4 ? 0xFF800000u
                     : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}

// The j-th value of a vector.
template <typename T>
__device__ __forceinline__ float pick(const uint4& raw, int j) {
  const int at = sizeof(T) == 4 ? j : j >> 1;
  const uint32_t w = at < 2 ? (at == 0 ? raw.x : raw.y) : (at == 2 ? raw.z : raw.w);
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const uint16_t h = uint16_t(j & 1 ? w >> 16 : w);
    if constexpr (std::is_same<T, __half>::value)
      return __half2float(__ushort_as_half(h));
    else
      return bf16_to_f32(h);
  }
}

// A row as slots of neighbouring columns: the columns before the first 16-byte
// boundary, the vectors, the columns after the last.
template <typename T>
struct Slots {
  static constexpr int kN = Vec16<T>::kN;
  const T* row;
  int head, vecs, tail;
  __device__ __forceinline__ Slots(const T* r, int n) : row(r) {
    const int off = int((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    head = min(n, off ? kN - off : 0);
    vecs = (n - head) / kN;
    tail = n - head - vecs * kN;
  }
  __device__ __forceinline__ const uint4* body() const {
    return reinterpret_cast<const uint4*>(row + head);
  }
  // slot s (0 .. vecs + 1): its values, first column and number
  __device__ __forceinline__ int get(int s, float (&f)[kN], int* col) const {
    if (s >= 1 && s <= vecs) {
      Vec16<T> v;
      v.raw = body()[s - 1];
      v.get(f);
      *col = head + (s - 1) * kN;
      return kN;
    }
    const int count = s == 0 ? head : s == vecs + 1 ? tail : 0;
    *col = s == 0 ? 0 : head + vecs * kN;
    for (int i = 0; i < kN; ++i) f[i] = i < count ? to_f32(row[*col + i]) : 0.f;
    return count;
  }
};

// Exact selection by radix passes over the whole row; fills sh.cut with the k
// keys.
template <typename T, int THREADS>
__device__ __noinline__ void select_exact(TopShared<THREADS / 32>& sh, const Slots<T>& row, int k) {
  constexpr int kN = Vec16<T>::kN;
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t prefix = 0, mask = 0;
  unsigned int need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    auto count = [&](float v, bool on) {
      const uint32_t key = key_of(v);
      on = on && (key & mask) == prefix;
      const unsigned int who = __ballot_sync(0xffffffffu, on);
      if (on) {
        const unsigned int bin = (key >> shift) & 255u;
        int one;  // lanes of one digit (equal rows) count once
        __match_all_sync(who, bin, &one);
        if (!one)
          atomicAdd(&sh.hist[bin], 1u);
        else if (lane == __ffs(who) - 1)
          atomicAdd(&sh.hist[bin], __popc(who));
      }
      __syncwarp();
    };
    {
      const bool on = tid < row.head + row.tail;
      count(on ? to_f32(row.row[tid < row.head ? tid : tid + row.vecs * kN]) : 0.f, on);
    }
    for (int i0 = 0; i0 < row.vecs; i0 += THREADS * kTopUnroll) {
      Vec16<T> v[kTopUnroll];
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
        const int i = i0 + u * THREADS + tid;
        v[u].raw = i < row.vecs ? row.body()[i] : lowest_vec<T>();
      }
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
#pragma unroll 1
        for (int j = 0; j < kN; ++j) count(pick<T>(v[u].raw, j), i0 + u * THREADS + tid < row.vecs);
      }
    }
    __syncthreads();
    if (tid == 0) {
      unsigned int above = 0;
      int bin = 255;
      while (bin > 0 && above + sh.hist[bin] < need) above += sh.hist[bin--];
      sh.digit = bin;
      sh.above = above;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    mask |= 255u << shift;
    need -= sh.above;  // of the values with this prefix
    __syncthreads();
  }
  // prefix is the k-th key; `need` of the values equal to it, by lowest column
  if (tid == 0) sh.kept = 0;
  __syncthreads();
  unsigned int equal_before = 0;
  const int slots = row.vecs + 2;
  for (int s0 = 0; s0 < slots; s0 += THREADS) {
    float f[kN];
    int col;
    const int count = row.get(s0 + tid, f, &col);
    int same = 0;
#pragma unroll
    for (int j = 0; j < kN; ++j) same += j < count && key_of(f[j]) == prefix ? 1 : 0;
    int upto = same;  // inclusive sum over the warp's lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sh.warp_sum[tid >> 5] = upto;
    __syncthreads();
    unsigned int before = equal_before + upto - same, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < tid >> 5) before += sh.warp_sum[w];
      total += sh.warp_sum[w];
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const uint32_t key = key_of(f[j]);
      const bool equal = j < count && key == prefix;
      if ((j < count && key > prefix) || (equal && before < need))
        sh.cut[atomicAdd(&sh.kept, 1)] = full_key(f[j], col + j);
      before += equal ? 1 : 0;
    }
    equal_before += total;
    __syncthreads();
  }
}

struct TopArgs {
  const void* logits;
  int64_t ld;
  int n, k, parts, each;
  float* values;
  int64_t* indices;
};

template <typename T, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) topk_kernel(const __grid_constant__ TopArgs g) {
  __shared__ TopShared<THREADS / 32> sh;
  constexpr int kN = Vec16<T>::kN;
  constexpr int kWarps = THREADS / 32;
  constexpr int kStep = THREADS * kTopUnroll;
  static_assert(THREADS % 32 == 0 && kWarps <= 8, "whole warps, slots for eight");
  const int tid = threadIdx.x;
  const int rank = g.parts > 1 ? int(cluster_rank()) : 0;
  const int64_t r = blockIdx.x / g.parts;
  const Slots<T> row(static_cast<const T*>(g.logits) + r * g.ld, g.n);
  const uint4* body = row.body();
  // this CTA's vectors; rank 0 takes the columns outside the vectors too
  const int v0 = int(int64_t(row.vecs) * rank / g.parts);
  const int v1 = int(int64_t(row.vecs) * (rank + 1) / g.parts);
  if (tid == 0) sh.kept = 0;
  const int warp = tid >> 5, lane = tid & 31;
  unsigned long long* mine = sh.list + warp * kTopWarpList;
  int listed = 0;                   // of this warp
  uint32_t first = 0, second = 0;   // this thread's largest maxima, as keys
  float floor_v = -INFINITY;
  // A value is listed unless it is below `bar`.  That is F, until this warp has
  // counted k values equal to F: it meets the columns in ascending order, so a
  // later one cannot be needed, and `bar` goes to the next value above F.  They
  // are counted where they come in numbers only.
  float bar = -INFINITY;
  int ties = 0;
  const int many = max(96, g.k + g.k / 2);  // listed: rows in no special order list fewer
  auto seen = [&](float m) {
    const uint32_t key = key_of(m);
    second = max(second, min(first, key));
    first = max(first, key);
  };
  auto refresh = [&]() {
    const uint32_t key = floor_of<kWarps>(first, second, g.each, sh.part);
    const float v = value_of(key);
    if (!(v == floor_v)) {
      floor_v = bar = v;
      ties = 0;
    }
    return key;
  };
  // the warp's lanes hold a value each, where `on`
  auto list = [&](float v, int col, bool on) {
    const unsigned int who = __ballot_sync(0xffffffffu, on);
    const int at = listed + __popc(who & ((1u << lane) - 1u));
    if (on && at < kTopWarpList) mine[at] = full_key(v, col);
    listed += __popc(who);
  };
  int loose_col = -1;
  float loose = 0.f;
  if (rank == 0 && tid < row.head + row.tail) {
    loose_col = tid < row.head ? tid : tid + row.vecs * kN;
    loose = to_f32(row.row[loose_col]);
    seen(loose);
  }
  // every thread goes through the same number of steps; past its vectors it
  // has nothing to look over
  const int steps = max(1, (v1 - v0 + kStep - 1) / kStep);
  int next = 0;  // the step at which F is refreshed
  auto load = [&](Vec16<T>(&v)[kTopUnroll], int step) {
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      const int i = v0 + step * kStep + u * THREADS + tid;
      v[u].raw = i < v1 ? __ldcs(body + i) : lowest_vec<T>();
    }
  };
  Vec16<T> v[kTopUnroll], ahead[kTopUnroll];
  load(v, 0);
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    if (step + 1 < steps) load(ahead, step + 1);
    const int at = v0 + step * kStep + tid;
    const float top = step_max<T>(v);
    if (step == 0) {  // the first bound from every vector's maximum
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u)
        if (at + u * THREADS < v1) seen(vec_max<T>(v[u]));
    } else if (at < v1) {
      seen(top);
    }
    if (step == next) {
      refresh();
      next = 2 * step + 1;
    }
    // out of order: these do not count as ties
    if (step == 0) list(loose, loose_col, loose_col >= 0 && !(loose < bar));
    if (__any_sync(0xffffffffu, !(top < bar))) {
      uint32_t take = not_below<T>(v, bar);
      if (step + 1 == steps) {  // vectors past the row's
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u)
          if (at + u * THREADS >= v1) take &= ~(0x000F000Fu << (4 * u));
      }
      if (listed > many || int(__reduce_add_sync(0xffffffffu, __popc(take))) > g.k - ties) {
        // perhaps more equal to F than needed: column by column
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u) {
          unsigned int here = 0;  // this vector's, in the columns' order
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const int b = sizeof(T) == 4 ? 4 * u + j : 4 * u + j / 2 + j % 2 * 16;
            here |= (take >> b & 1u) << j;
          }
          unsigned int same = 0;
#pragma unroll 1
          for (int j = 0; j < kN; ++j)
            same |= (here >> j & 1u) && pick<T>(v[u].raw, j) == floor_v ? 1u << j : 0u;
          int before = __popc(same);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += w;
          }
          const int equal = __shfl_sync(0xffffffffu, before, 31);
          before -= __popc(same);
          while (same && before + __popc(same) > g.k - ties) {  // the first columns' stay
            const unsigned int last = 1u << (31 - __clz(same));
            same ^= last;
            here ^= last;
          }
          ties += equal;  // this warp's later columns are above these
          if (ties > g.k) ties = g.k;
          while (__any_sync(0xffffffffu, here)) {  // each lane's lowest remaining one
            const int j = __ffs(here) - 1;
            list(pick<T>(v[u].raw, j & (kN - 1)), row.head + (at + u * THREADS) * kN + j, here != 0);
            here &= here - 1;
          }
        }
        if (ties >= g.k && floor_v < INFINITY) bar = nextafterf(floor_v, INFINITY);
      } else {
        while (__any_sync(0xffffffffu, take)) {  // one of each lane's
          int col;
          const float x = value_at<T>(v, __ffs(take) - 1, THREADS * kN, &col);
          list(x, row.head + at * kN + col, take != 0);
          take &= take - 1;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) v[u] = ahead[u];
  }
  if (lane == 0) sh.listed[warp] = listed;
  uint32_t floor_key = refresh();
  // settled: the refresh's barriers follow the last append
  bool over = false;
  for (int i = 0; i < kWarps; ++i) over |= sh.listed[i] > kTopWarpList;
  if (g.parts > 1) {
    if (tid == 0) {
      sh.floor_key = floor_key;
      sh.over = over;
    }
    __syncwarp();
    cluster_sync_all();
    // a lane per CTA: one remote access after another would cost as many latencies
    const int from = lane < g.parts ? lane : 0;
    const uint32_t theirs = ld_cluster_u32(map_rank(smem_u32(&sh.floor_key), from));
    over = ld_cluster_u32(map_rank(smem_u32(&sh.over), from)) != 0;
    floor_key = __reduce_max_sync(0xffffffffu, theirs);
    over = __any_sync(0xffffffffu, over);
  }
  if (!over) {
    for (int i = lane; i < listed; i += 32) {
      const unsigned long long key = mine[i];
      if (uint32_t(key >> 32) >= floor_key) {
        const int at = atomicAdd(&sh.kept, 1);
        if (at < kTopShort) sh.cut[at] = key;
      }
    }
  }
  __syncthreads();
  const unsigned long long* all = sh.cut;
  int kept = sh.kept, total = kept;
  if (g.parts == 1) {
    over |= kept > kTopShort;
    __syncthreads();
  } else {
    __syncwarp();
    cluster_sync_all();  // every CTA's survivors are in place
    const int theirs =
        lane < g.parts ? int(ld_cluster_u32(map_rank(smem_u32(&sh.kept), lane))) : 0;
    over |= __any_sync(0xffffffffu, theirs > kTopShort);
    int end[8];  // of each CTA's survivors in the joint list
    total = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) end[i] = total += __shfl_sync(0xffffffffu, theirs, i);
    over |= total > sh.kList;
    if (!over) {
      for (int at = tid; at < total; at += THREADS) {
        int from = 0, start = 0;
#pragma unroll
        for (int i = 0; i < 7; ++i) {
          if (at >= end[i]) {
            from = i + 1;
            start = end[i];
          }
        }
        sh.list[at] = ld_cluster_u64(map_rank(smem_u32(sh.cut), from) + uint32_t(at - start) * 8u);
      }
      all = sh.list;
    }
    // the survivors have been read: they may be written again, or the CTA leave
    __syncwarp();
    cluster_sync_all();
    __syncthreads();
  }
  if (over) {  // the same in the whole cluster
    if (rank != 0) return;
    select_exact<T, THREADS>(sh, row, g.k);
    __syncthreads();
    kept = total = sh.kept;
  }
  for (int i = tid; i < kept; i += THREADS) {
    const unsigned long long key = sh.cut[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < total; ++j) place += all[j] > key ? 1 : 0;
    if (place < g.k) {
      g.values[r * g.k + place] = value_of(uint32_t(key >> 32));
      g.indices[r * g.k + place] = 0x7FFFFFFF - int(uint32_t(key));
    }
  }
}

template <typename T, int THREADS, int CTAS>
int launch_topk(TopArgs g, int64_t rows, int parts, cudaStream_t stream) {
  g.parts = parts;
  g.each = (g.k + THREADS / 32 - 1) / (THREADS / 32);
  if (rows * parts > 0x7fffffff) return MR_ERR_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, topk_kernel<T, THREADS, CTAS>, g);
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

extern "C" int mr_topk_logits(const void* logits, int64_t rows, int n, int64_t ld, int k, int dtype,
                              float* values, int64_t* indices, void* stream) {
  if (!logits || !values || !indices || rows <= 0 || rows > 0x7fffffff || n <= 0 || k <= 0 ||
      k > kTopMaxK || k > n || ld < n || !known_dtype(dtype))
    return MR_ERR_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(logits) % elt_bytes(dtype)) return MR_ERR_ALIGNMENT;
  TopArgs g;
  g.logits = logits;
  g.ld = ld;
  g.n = n;
  g.k = k;
  g.values = values;
  g.indices = indices;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t row_bytes = int64_t(n) * elt_bytes(dtype);
  // few rows are divided, down to shares of 16 KB
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * sm_count() && row_bytes / (parts * 2) >= 16384)
    parts *= 2;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    // short rows: smaller blocks, more rows per SM and no idle threads (up to
    // 32 of the k per warp)
    if (row_bytes <= 16384 && k <= 128) return launch_topk<T, 128, 8>(g, rows, 1, st);
    return launch_topk<T, 256, 4>(g, rows, parts, st);
  });
}
