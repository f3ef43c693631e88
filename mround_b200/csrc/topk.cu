// K11 -- the k largest values of each row, with their columns.
//
// Order: larger value first, NaN above everything, equal values (and +0 / -0)
// by lowest column.  HBM-bound: a row is read once.
//
// One block per row streams it with 16-byte loads and keeps a lower bound T of
// the k-th largest value: each thread keeps the maximum of what it has seen,
// the threads form G >= k disjoint groups, and T is the smallest of the groups'
// maxima -- every group holds a value >= T, so at least k values are >= T and
// what is below T cannot be among the k largest.  Values not below T go to a
// list in shared memory.  T is refreshed when the part read has doubled, so a
// row in no special order lists about G ln G values per doubling.  At the end
// the list is cut to the last T and each survivor's rank is the number of
// listed keys above it (value, then column: all keys differ), which is also its
// place in the output: no sort.
//
// A row whose list overflows (long runs of equal values, a fully masked row, a
// rising row) takes the exact way instead: four 8-bit radix passes over the row
// (from L2) find the k-th key and the number above it; the values above it, and
// the first columns equal to it, form the list.
//
// Results do not depend on the order in which threads append to the list.

#include <type_traits>

#include "rowtypes.cuh"
#include "sm100.cuh"

namespace mr {
namespace {

constexpr int kTopThreads = 512;
constexpr int kTopUnroll = 4;     // 16-byte loads in flight per thread
constexpr int kTopList = 6144;    // listed values while streaming
constexpr int kTopShort = 2048;   // of them, not below the last T
constexpr int kTopMaxK = 256;     // groups of at least two threads

struct TopShared {
  unsigned long long list[kTopList];
  unsigned long long cut[kTopShort];
  unsigned int hist[256];
  float part[kTopThreads / 32];
  int listed, kept, warp_sum[kTopThreads / 32];
  unsigned int digit, above;
};

// Order-preserving 32-bit key; NaN is the largest, -0 equals +0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  if (v == 0.f) v = 0.f;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __int_as_float(0x7fffffff);
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ unsigned long long full_key(float v, int col) {
  return (static_cast<unsigned long long>(key_of(v)) << 32) | uint32_t(0x7FFFFFFF - col);
}

// The smallest of the groups' maxima, to every thread (group: `per` lanes).
__device__ __forceinline__ float group_floor(float m, int per, float* part) {
  for (int o = per >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fminf(m, __shfl_xor_sync(0xffffffffu, m, o));
  __syncthreads();  // the last reader of part is done
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  float all = part[threadIdx.x & (kTopThreads / 32 - 1)];
#pragma unroll
  for (int o = kTopThreads / 64; o > 0; o >>= 1)
    all = fminf(all, __shfl_xor_sync(0xffffffffu, all, o));
  return all;
}

__device__ __forceinline__ void list_value(TopShared& sh, float v, int col) {
  const int at = atomicAdd(&sh.listed, 1);
  if (at < kTopList) sh.list[at] = full_key(v, col);
}

// Exact selection by radix passes; fills sh.cut with the k keys.
template <typename T>
__device__ void select_exact(TopShared& sh, const T* row, int n, int k) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0, mask = 0;
  unsigned int need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kTopThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kTopThreads) {
      const int i = i0 + tid;
      const uint32_t key = i < n ? key_of(to_f32(row[i])) : 0;
      const bool on = i < n && (key & mask) == prefix;
      const unsigned int who = __ballot_sync(0xffffffffu, on);
      if (!on) continue;
      // lanes with one digit in common (equal rows) count once per warp
      const unsigned int bin = (key >> shift) & 255u;
      const unsigned int peers = __match_any_sync(who, bin);
      if ((tid & 31) == __ffs(peers) - 1) atomicAdd(&sh.hist[bin], __popc(peers));
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
  for (int i0 = 0; i0 < n; i0 += kTopThreads) {
    const int i = i0 + tid;
    const float v = i < n ? to_f32(row[i]) : 0.f;
    const uint32_t key = i < n ? key_of(v) : 0;
    const bool same = i < n && key == prefix;
    const unsigned int votes = __ballot_sync(0xffffffffu, same);
    if ((tid & 31) == 0) sh.warp_sum[tid >> 5] = __popc(votes);
    __syncthreads();
    unsigned int before = equal_before, total = 0;
    for (int w = 0; w < kTopThreads / 32; ++w) {
      if (w < tid >> 5) before += sh.warp_sum[w];
      total += sh.warp_sum[w];
    }
    before += __popc(votes & ((1u << (tid & 31)) - 1u));
    if ((i < n && key > prefix) || (same && before < need))
      sh.cut[atomicAdd(&sh.kept, 1)] = full_key(v, i);
    equal_before += total;
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 3)
    topk_kernel(const T* __restrict__ logits, int64_t ld, int n, int k, int per,
                float* __restrict__ values, int64_t* __restrict__ indices) {
  extern __shared__ __align__(16) uint8_t raw[];
  TopShared& sh = *reinterpret_cast<TopShared*>(raw);
  constexpr int kN = Vec16<T>::kN;
  const int tid = threadIdx.x;
  const T* row = logits + int64_t(blockIdx.x) * ld;
  // columns before the first 16-byte boundary, and after the last
  const int off = int((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int head = min(n, off ? kN - off : 0);
  const int vecs = (n - head) / kN;
  const int loose = n - vecs * kN;  // head and tail columns
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  if (tid == 0) {
    sh.listed = 0;
    sh.kept = 0;
  }
  float best = -INFINITY, odd = -INFINITY;
  int odd_col = -1;
  if (tid < loose) {
    odd_col = tid < head ? tid : tid + vecs * kN;
    odd = to_f32(row[odd_col]);
    best = odd;
  }
  float floor_v = -INFINITY;
  int refresh = 0;
  for (int c = 0; c * kTopThreads * kTopUnroll < vecs || c == 0; ++c) {
    Vec16<T> v[kTopUnroll];
    const int first = c * kTopThreads * kTopUnroll + tid;
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u)
      if (first + u * kTopThreads < vecs) v[u].raw = __ldg(body + first + u * kTopThreads);
    float m[kTopUnroll];
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      m[u] = -INFINITY;
      if (first + u * kTopThreads < vecs) {
        float f[kN];
        v[u].get(f);
        bool nan = false;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          m[u] = fmaxf(m[u], f[j]);
          nan |= f[j] != f[j];
        }
        best = fmaxf(best, m[u]);
        if (nan) m[u] = __int_as_float(0x7fffffff);
      }
    }
    if (c == refresh) {
      floor_v = group_floor(best, per, sh.part);
      refresh = 2 * c + 1;
    }
    if (c == 0 && odd_col >= 0 && !(odd < floor_v)) list_value(sh, odd, odd_col);
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      if (first + u * kTopThreads < vecs && !(m[u] < floor_v)) {
        float f[kN];
        v[u].get(f);
        const int col = head + (first + u * kTopThreads) * kN;
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (!(f[j] < floor_v)) list_value(sh, f[j], col + j);
      }
    }
  }
  floor_v = group_floor(best, per, sh.part);
  const uint32_t floor_key = key_of(floor_v);
  const int listed = sh.listed;  // settled: group_floor's barriers follow the last append
  bool exact = listed > kTopList;
  if (!exact) {
    for (int i = tid; i < listed; i += kTopThreads) {
      const unsigned long long key = sh.list[i];
      if (uint32_t(key >> 32) >= floor_key) {
        const int at = atomicAdd(&sh.kept, 1);
        if (at < kTopShort) sh.cut[at] = key;
      }
    }
    __syncthreads();
    exact = sh.kept > kTopShort;
    __syncthreads();
  }
  if (exact) select_exact(sh, row, n, k);
  __syncthreads();
  const int kept = sh.kept;
  for (int i = tid; i < kept; i += kTopThreads) {
    const unsigned long long key = sh.cut[i];
    int rank = 0;
    for (int j = 0; j < kept; ++j) rank += sh.cut[j] > key ? 1 : 0;
    if (rank < k) {
      values[int64_t(blockIdx.x) * k + rank] = value_of(uint32_t(key >> 32));
      indices[int64_t(blockIdx.x) * k + rank] = 0x7FFFFFFF - int(uint32_t(key));
    }
  }
}

template <typename T>
int launch_topk(const void* logits, int64_t rows, int n, int64_t ld, int k, float* values,
                int64_t* indices, cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices];
  const int status = raise_smem(topk_kernel<T>, int(sizeof(TopShared)), configured);
  if (status != MR_OK) return status;
  int groups = 32;
  while (groups < k) groups *= 2;
  topk_kernel<T><<<unsigned(rows), kTopThreads, sizeof(TopShared), stream>>>(
      static_cast<const T*>(logits), ld, n, k, kTopThreads / groups, values, indices);
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
  return with_dtype(dtype, [&](auto tag) {
    return launch_topk<decltype(tag)>(logits, rows, n, ld, k, values, indices,
                                      static_cast<cudaStream_t>(stream));
  });
}
