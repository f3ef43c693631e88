// K13 -- matrix product with bias, activation and residual in its epilogue,
// on the tcgen05 tensor cores (sm_100a).
//
//   z[t, f] = sum_k x[t, k] w[f, k] + bias[f]
//   y = act(z)  (none, SiLU, GELU by erf or tanh; SwiGLU: the features are
//   [gate | up] and y = silu(z_gate) z_up)      out = y + residual
//
// Operands are bf16, each either one tensor or a hi/lo pair (x = hi + lo), as
// in K3: one, two (x a pair) or three (both pairs) products into one float32
// accumulator, per 16 k in the order x_hi w_hi, x_hi w_lo, x_lo w_hi.  Either
// operand may be K-major or MN-major, which makes the two gradient products of
// a linear the same kernel.
//
// The features are the MMA's M and the tokens its N.  An accumulator lane is
// then one feature: the bias is one register per thread, a warp's store is 32
// neighbouring features of one token, and N shrinks with the tokens (16 for a
// single one) while the weights keep all 128 lanes busy -- few tokens cost one
// reading of the weights.  SwiGLU takes 64 gate rows and the 64 up rows of the
// same features into one 128-row tile.
//
// split kernel: one tile of 128 features x BT tokens per CTA, K divided among
// the CTAs of a cluster.  Each leaves its float32 partial tile in its own
// shared memory; the cluster's CTAs then each finish a share of the tokens,
// reading the partials over distributed shared memory in rank order, so the
// result does not depend on timing and needs no workspace.
//
// Roles (256 threads): warps 0 and 6 TMA producers (features, tokens); warp 1
// TMEM and MMA issuer; warps 2-5 read the accumulator; all finish the outputs.
// Producers and issuer run as whole warps with one elected lane, so that their
// operands stay in uniform registers, and look at the next stage's barrier
// before they issue this one's work.
// Every mbarrier wait is bounded: one that gives up sets the status word that
// mr_gemm_status reads, and every role goes on to the barriers at the end.

#include <string.h>

#include <algorithm>
#include <cmath>

#include "linear.h"
#include "rowtypes.cuh"
#include "sm100.cuh"

namespace mr {
namespace {

constexpr int kBK = 64;                // K per stage: 128-byte rows
constexpr int kTileF = 128;            // accumulator lanes per CTA
constexpr int kABytes = kTileF * kBK * 2;
constexpr uint64_t kWaitLimitNs = 2000000000ull;  // 2 s per wait

__device__ int g_linear_status = 0;

// Bounded wait; returns false (and raises the status word) on timeout.  The
// clock is read only after many tries: reading it costs as much as a stage.
__device__ __forceinline__ bool lin_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 1024; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u) {
      if (globaltimer() - t0 > kWaitLimitNs) {
        atomicExch(&g_linear_status, MR_ERR_TIMEOUT);
        return false;
      }
      if (*reinterpret_cast<volatile int*>(&g_linear_status) != 0) return false;
    }
  }
}

// The same by a whole warp, whose lanes go on together.
__device__ __forceinline__ bool lin_wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, lin_wait(bar, parity));
}

// Whether the phase is complete, without waiting.
__device__ __forceinline__ bool lin_peek(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A ring position: stage and the parity of its current use.
struct Ring {
  int s = 0;
  uint32_t phase;
  __device__ __forceinline__ explicit Ring(uint32_t p) : phase(p) {}
  template <int kStages>
  __device__ __forceinline__ void next() {
    if (++s == kStages) {
      s = 0;
      phase ^= 1;
    }
  }
};

// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

struct LinMaps {
  CUtensorMap a_hi, a_lo, b_hi, b_lo;  // a: features, b: tokens
  int a_kmajor, b_kmajor;
};

template <int PREC>
__device__ __forceinline__ void prefetch_maps(const LinMaps& m) {
  auto fetch = [](const CUtensorMap* p) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(p)) : "memory");
  };
  fetch(&m.a_hi);
  fetch(&m.b_hi);
  if (PREC == 3) fetch(&m.a_lo);
  if (PREC >= 2) fetch(&m.b_lo);
}

// What follows the product.  feats counts outputs (half of the features under
// SwiGLU, whose up rows start at row `feats`).
struct LinEpilogue {
  const float* bias;
  const void* residual;
  void* out;
  uint16_t* lo;
  float* t32;
  float* pre;
  int64_t ldr, ldo, ldp;
  int residual_dtype, out_dtype, act, feats, toks;
};

// silu as the block's element-wise kernels compute it
__device__ __forceinline__ float silu1(float g) { return g / (1.f + expf(-g)); }

// The activations for a bf16 result, without the exact division's branches: to
// 2^-20 of |z|, and to 2^-13 of the value where that is smaller.  The branches,
// unrolled over 32 tokens, made the epilogue longer than the products: 2047 x
// 2048 by 11008 features take 92 us with an exactly divided tanh GELU, 70 us so,
// 66 us without an activation.  Float32 results, and pairs, take the exact forms.
__device__ __forceinline__ float silu_rough(float g) {
  return __fdividef(g, 1.f + __expf(-g));
}

// Phi(-|z|) = t 2^(p(t) - z^2 log2(e) / 2), t = 1 / (1 + |z| / 2): the form of
// erfc's Chebyshev fit in Press et al., Numerical Recipes (2nd edition, 6.2).  p
// is our own fit, of degree 8 and least largest error for |z| <= 13.2, where the
// tail leaves float32's range: 6.4e-7 of the tail with these rounded constants.
__device__ __forceinline__ float gelu_tail(float z) {
  const float t = __fdividef(1.f, fmaf(0.5f, fabsf(z), 1.f));
  float p = fmaf(0.102767207f, t, -0.193010613f);
  p = fmaf(p, t, -0.514969468f);
  p = fmaf(p, t, 1.905410767f);
  p = fmaf(p, t, -1.959707379f);
  p = fmaf(p, t, 0.271629959f);
  p = fmaf(p, t, 0.261255383f);
  p = fmaf(p, t, 1.452787995f);
  p = fmaf(p, t, -2.326163054f);
  float power;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(fmaf(-0.72134752f * z, z, p)));
  return t * power;
}

__device__ __forceinline__ float gelu_rough(float z) {
  const float tail = gelu_tail(z);
  return z * (z < 0.f ? tail : 1.f - tail);
}

// (1 + tanh u) / 2 = 1 / (1 + e^-2u)
__device__ __forceinline__ float gelu_tanh_arg(float z) {
  return -1.5957691216057308f * (z + 0.044715f * z * z * z);
}
__device__ __forceinline__ float gelu_tanh_rough(float z) {
  return __fdividef(z, 1.f + __expf(gelu_tanh_arg(z)));
}

template <int N>
__device__ __forceinline__ void activate(int act, bool rough, float (&v)[N]) {
  auto each = [&](auto fn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fn(v[i]);
  };
  if (act == MR_ACT_SILU) {
    if (rough)
      each(silu_rough);
    else
      each(silu1);
  } else if (act == MR_ACT_GELU) {
    if (rough)
      each(gelu_rough);
    else
      each([](float z) { return 0.5f * z * (1.f + erff(z * 0.70710678118654752f)); });
  } else if (act == MR_ACT_GELU_TANH) {
    if (rough)
      each(gelu_tanh_rough);
    else
      each([](float z) { return z / (1.f + expf(gelu_tanh_arg(z))); });
  }
}

// The epilogue of tokens t0 .. t0 + N - 1, as far as `end`, of one feature: v
// holds z (up: the up row's).
template <bool kGated, int N>
__device__ __forceinline__ void finish_run(const LinEpilogue& e, int f, int t0, int end,
                                           float (&v)[N], const float (&up)[N]) {
  if (f >= e.feats || t0 >= end) return;
  const bool rough = e.out_dtype == MR_BF16 && !e.lo;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!kGated) break;
    v[i] = (rough ? silu_rough(v[i]) : silu1(v[i])) * up[i];
  }
  if (!kGated) activate(e.act, rough, v);
  auto store = [&](auto whole) {  // whole: all N tokens exist
    constexpr bool kWhole = decltype(whole)::value;
    const int n = kWhole ? N : end - t0;
    if (e.residual) {
      float r[N];
      if (e.residual_dtype == MR_F32) {
        const float* p = static_cast<const float*>(e.residual) + int64_t(t0) * e.ldr + f;
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = kWhole || i < n ? p[i * e.ldr] : 0.f;
      } else {
        const uint16_t* p = static_cast<const uint16_t*>(e.residual) + int64_t(t0) * e.ldr + f;
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = kWhole || i < n ? bf16_to_f32(p[i * e.ldr]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += r[i];
    }
    const int64_t at = int64_t(t0) * e.ldo + f;
    if (e.out_dtype == MR_F32) {
      float* p = static_cast<float*>(e.out) + at;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (kWhole || i < n) p[i * e.ldo] = v[i];
    } else {
      uint16_t* p = static_cast<uint16_t*>(e.out) + at;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (kWhole || i < n) p[i * e.ldo] = f32_to_bf16(v[i]);
      if (e.lo) {
        uint16_t* l = e.lo + at;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (kWhole || i < n)
            l[i * e.ldo] = f32_to_bf16(__fsub_rn(v[i], bf16_to_f32(f32_to_bf16(v[i]))));
      }
    }
    if (e.t32) {
      float* p = e.t32 + at;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (kWhole || i < n) p[i * e.ldo] = tf32_rna(v[i]);
    }
  };
  if (t0 + N <= end)
    store(std::true_type());
  else
    store(std::false_type());
}

// Stores z of tokens t0 .. t0 + N - 1, as far as `end`, for one row of w.
template <int N>
__device__ __forceinline__ void store_pre(const LinEpilogue& e, int row, bool on, int t0, int end,
                                          const float (&v)[N]) {
  if (!on) return;
  float* p = e.pre + int64_t(t0) * e.ldp + row;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (t0 + i < end) p[i * e.ldp] = v[i];
}

// bf16 x bf16 -> float32
__host__ __device__ constexpr uint32_t lin_idesc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// Descriptors of 128-byte-swizzled tiles.  K-major: rows of 64 k, 8-row groups
// 1024 B apart, 16 k are 32 B.  MN-major: boxes of 64 columns x 64 k (8 KB),
// 8-k groups 1024 B apart, 16 k are 2048 B.  Only the address field (the low
// word's 14 bits, in 16 bytes) changes from one MMA to the next: the issuing
// thread adds to it, since building a descriptor per MMA took it as long as
// the MMAs (450 ns per stage whatever the tile's width).
struct LinDesc {
  uint32_t low, high, step;  // step: 16 k further
  __device__ __forceinline__ LinDesc(uint32_t base, bool kmajor) {
    const uint64_t d = kmajor ? smem_desc(base, 16, 1024, 2)
                              : smem_desc(base, 64 * kBK * 2, 1024, 2);
    low = uint32_t(d);
    high = uint32_t(d >> 32);
    step = kmajor ? 32 >> 4 : 2048 >> 4;
  }
  // the tile `bytes` further, ks * 16 k in
  __device__ __forceinline__ uint64_t at(uint32_t bytes16, int ks) const {
    return (uint64_t(high) << 32) | (low + bytes16 + step * ks);
  }
};

template <int BT, int PREC>
struct SplitCfg {
  static constexpr int kAParts = PREC == 3 ? 2 : 1;
  static constexpr int kBParts = PREC >= 2 ? 2 : 1;
  static constexpr int kBBytes = BT * kBK * 2;
  static constexpr int kStage = kABytes * kAParts + kBBytes * kBParts;
  // two CTAs per SM where four stages fit half of its shared memory
  static constexpr int kBudget = kStage * 4 <= 104 * 1024 ? 104 * 1024 : 208 * 1024;
  static constexpr int kStages = kBudget / kStage > 8 ? 8 : kBudget / kStage;
  static constexpr int kPartial = BT * kTileF * 4;  // reuses the stages
  static constexpr int kSmem = kStages * kStage + 1024 /* align */ + 256 /* barriers */;
  static constexpr int kTmemCols = BT < 32 ? 32 : BT;
  static_assert(kStages * kStage >= kPartial, "the partial tile must fit the stages");
};

constexpr int kSplitThreads = 256;

// One stage of a tile: features from f0 (SwiGLU: 64 gate rows and their up
// rows), tokens from t0, k from k0.
template <int ROWS>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                                          bool kmajor, int row0, int k0) {
  if (kmajor) {
    tma_load_3d(dst, map, bar, k0, row0, 0);
  } else {
#pragma unroll
    for (int c = 0; c < ROWS / 64; ++c)
      tma_load_3d(dst + c * 64 * kBK * 2, map, bar, row0 + c * 64, k0, 0);
  }
}

template <bool kGated>
__device__ __forceinline__ void load_features(uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                                              bool kmajor, int f0, int up0, int k0) {
  if constexpr (kGated) {
    tma_load_3d(dst, map, bar, k0, f0, 0);
    tma_load_3d(dst + kABytes / 2, map, bar, k0, up0 + f0, 0);
  } else {
    load_rows<kTileF>(dst, map, bar, kmajor, f0, k0);
  }
}

template <int BT, int PREC, bool kGated>
__global__ void __launch_bounds__(kSplitThreads)
    linear_split_kernel(const __grid_constant__ LinMaps maps,
                        const __grid_constant__ LinEpilogue e, int k, int splits, int f_tiles) {
  using C = SplitCfg<BT, PREC>;
  constexpr int kOut = kGated ? kTileF / 2 : kTileF;  // outputs per tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStage);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = splits > 1 ? int(cluster_rank()) : 0;
  const int tile = blockIdx.x / splits;
  const int f0 = (tile % f_tiles) * kOut, t0 = (tile / f_tiles) * BT;
  const int k_tiles = (k + kBK - 1) / kBK;
  const int per = (k_tiles + splits - 1) / splits;
  const int kt0 = min(rank * per, k_tiles), kt1 = min(kt0 + per, k_tiles);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 2);  // two producers
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_maps<PREC>(maps);
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 || warp == 6) {
    // features by warp 0, tokens by warp 6: one warp issuing both, a lane of its
    // own, took 300 ns per stage, this takes 175
    const bool leader = elect_one();
    Ring ring(1);  // of the stages' previous use; the first passes at once
    bool ready = false;
    for (int kt = kt0; kt < kt1; ++kt) {
      const int s = ring.s;
      if (!ready && !lin_wait_warp(&empty[s], ring.phase)) break;
      ring.next<C::kStages>();
      const bool peeked = lin_peek(&empty[ring.s], ring.phase);
      if (leader && warp == 0) {
        uint8_t* st = smem + s * C::kStage;
        mbar_expect_tx(&full[s], kABytes * C::kAParts);
        load_features<kGated>(st, &maps.a_hi, &full[s], maps.a_kmajor, f0, e.feats, kt * kBK);
        if constexpr (C::kAParts == 2)
          load_features<kGated>(st + kABytes, &maps.a_lo, &full[s], maps.a_kmajor, f0, e.feats,
                                kt * kBK);
      } else if (leader) {
        mbar_expect_tx(&full[s], C::kBBytes * C::kBParts);
        uint8_t* sb = smem + s * C::kStage + kABytes * C::kAParts;
        load_rows<BT>(sb, &maps.b_hi, &full[s], maps.b_kmajor, t0, kt * kBK);
        if constexpr (C::kBParts == 2)
          load_rows<BT>(sb + C::kBBytes, &maps.b_lo, &full[s], maps.b_kmajor, t0, kt * kBK);
      }
      ready = __all_sync(0xffffffffu, peeked);
    }
  } else if (warp == 1) {
    const uint32_t idesc = lin_idesc(128, BT, !maps.a_kmajor, !maps.b_kmajor);
    const LinDesc da(smem_u32(smem), maps.a_kmajor);
    const LinDesc db(smem_u32(smem) + kABytes * C::kAParts, maps.b_kmajor);
    const bool leader = elect_one();
    Ring ring(0);
    bool ready = false;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!ready && !lin_wait_warp(&full[ring.s], ring.phase)) break;
      const int s = ring.s;
      ring.next<C::kStages>();
      // looked at before this stage's MMAs go out, read after them
      const bool peeked = kt + 1 < kt1 && lin_peek(&full[ring.s], ring.phase);
      const uint32_t off = uint32_t(s) * (C::kStage >> 4);
      if (leader) {
#pragma unroll
        for (int ks = 0; ks < kBK / 16; ++ks) {
          const uint64_t dah = da.at(off, ks), dbh = db.at(off, ks);
          umma_bf16(tmem, dah, dbh, idesc, (kt > kt0 || ks > 0) ? 1u : 0u);
          if constexpr (PREC == 3) umma_bf16(tmem, da.at(off + (kABytes >> 4), ks), dbh, idesc, 1u);
          if constexpr (PREC >= 2)
            umma_bf16(tmem, dah, db.at(off + (C::kBBytes >> 4), ks), idesc, 1u);
        }
        umma_commit(&empty[s]);
      }
      ready = __all_sync(0xffffffffu, peeked);
    }
    if (leader) umma_commit(done);
  }
  __syncwarp();
  // every MMA of this CTA has completed: the accumulator may be read, and the
  // stages hold nothing that is still needed
  const bool ok = lin_wait(done, 0) && *reinterpret_cast<volatile int*>(&g_linear_status) == 0;
  tc_fence_after();
  float* partial = reinterpret_cast<float*>(smem);  // [token][lane]
  const int toks = min(BT, e.toks - t0);
  if (warp >= 2 && warp < 6 && __all_sync(0xffffffffu, ok)) {
    const int quarter = warp & 3;
    const int f = quarter * 32 + lane;
    constexpr int kCols = BT < 32 ? 32 : BT;
#pragma unroll 1
    for (int col = 0; col < kCols && col < toks; col += 32) {
      float v[32];
      __syncwarp();
      tmem_ld32(tmem + (uint32_t(quarter * 32) << 16) + col, v);
#pragma unroll
      for (int q = 0; q < 32; ++q)
        if (col + q < toks) partial[(col + q) * kTileF + f] = kt1 > kt0 ? v[q] : 0.f;
    }
  }
  tc_fence_before();
  __syncwarp();
  if (splits > 1) cluster_sync_all(); else __syncthreads();
  if (ok) {
    // each thread a feature and runs of kRun tokens, loaded together
    constexpr int kRun = BT >= 64 ? 8 : 4;
    const int share = ((toks + splits - 1) / splits + kRun - 1) / kRun * kRun;
    const int first = rank * share, last = min(first + share, toks);
    const int f = threadIdx.x % kOut;
    const uint32_t base = smem_u32(partial) + uint32_t(f) * 4u;
    const bool on = f0 + f < e.feats;
    float bias = 0.f, bias_up = 0.f;
    if (e.bias && on) {
      bias = e.bias[f0 + f];
      if (kGated) bias_up = e.bias[e.feats + f0 + f];
    }
    for (int t = first + int(threadIdx.x) / kOut * kRun; t < last;
         t += kSplitThreads / kOut * kRun) {
      float z[kRun] = {}, zu[kRun] = {};
      for (int s = 0; s < splits; ++s) {
        // plain loads of this CTA's own memory where nothing is divided
        const uint32_t from = (splits > 1 ? map_rank(base, s) : base) + uint32_t(t * kTileF) * 4u;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          if (t + i < last) {
            z[i] += ld_cluster(from + uint32_t(i * kTileF) * 4u);
            if (kGated) zu[i] += ld_cluster(from + uint32_t(i * kTileF + kOut) * 4u);
          }
        }
      }
      if (e.bias) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          z[i] += bias;
          if (kGated) zu[i] += bias_up;
        }
      }
      if (e.pre) {
        store_pre(e, f0 + f, on, t0 + t, t0 + last, z);
        if (kGated) store_pre(e, e.feats + f0 + f, on, t0 + t, t0 + last, zu);
      }
      finish_run<kGated, kRun>(e, f0 + f, t0 + t, t0 + last, z, zu);
    }
  }
  if (!ok) {  // let issued copies land before the CTA exits
    const uint64_t t = globaltimer();
    while (globaltimer() - t < 1000000ull) {
    }
  }
  // no CTA leaves while another may still read its partial tile
  __syncwarp();
  if (splits > 1) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}


// ---------------------------------------------------------------- wide kernel
// Many tokens: a persistent kernel of CTA pairs.  A pair computes 256 features
// x BT tokens (256, or fewer where that shortens the schedule) with
// tcgen05.mma.cta_group::2 (M = 256, N = BT): each CTA stages its 128 feature
// rows and half of the token rows and keeps its 128 lanes x BT columns of the
// accumulator, so a stage holds 256 rows of k for 2 x 128 x 256 flops per k and
// CTA -- a third less than a 128 x 256 tile of one CTA.  Two accumulators: the
// epilogue of one tile, by eight warps (SiLU's exponential and division took
// four warps as long as the MMAs of k = 3584), overlaps the MMAs of the next.
//
// The leader (rank 0) issues the MMAs for both.  Both CTAs' loads complete on
// the leader's "full" barrier; the MMAs' commits free the stage, and publish
// the accumulator, on the barriers of both; the epilogue warps of both arrive
// on the leader's "tmem_empty".
constexpr int kWideThreads = 320;
constexpr int kWideT = 256;          // most tokens per tile
constexpr int kWideBufs = 2;         // accumulators of 256 columns

template <int PREC>
struct WideCfg {
  static constexpr int kAParts = PREC == 3 ? 2 : 1;
  static constexpr int kBParts = PREC >= 2 ? 2 : 1;
  static constexpr int kBBytes = kWideT / 2 * kBK * 2;
  static constexpr int kStage = kABytes * kAParts + kBBytes * kBParts;
  static constexpr int kStages = 192 * 1024 / kStage;
  // SwiGLU: two buffers of 16 x 32 float32 in each direction per pair of warps
  static constexpr int kExchange = 4 * 2 * 2 * 16 * 32 * 4;
  static constexpr int kSmem = kStages * kStage + kExchange + 1024 /* align */ + 256;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                              int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(0)
      : "memory");
}

// One operand part of a stage: rows as high as the map's box (K-major), or
// `chunks` of 64 rows (MN-major).
__device__ __forceinline__ void load_pair_rows(uint8_t* dst, const CUtensorMap* map, uint32_t bar,
                                               bool kmajor, int row0, int k0, int chunks) {
  if (kmajor) {
    tma_load_pair(dst, map, bar, k0, row0);
  } else {
    for (int c = 0; c < chunks; ++c)
      tma_load_pair(dst + c * 64 * kBK * 2, map, bar, row0 + c * 64, k0);
  }
}

template <bool kGated>
__device__ __forceinline__ void load_pair_features(uint8_t* dst, const CUtensorMap* map,
                                                   uint32_t bar, bool kmajor, int f0, int up0,
                                                   int k0) {
  if constexpr (kGated) {
    tma_load_pair(dst, map, bar, k0, f0);
    tma_load_pair(dst + kABytes / 2, map, bar, k0, up0 + f0);
  } else {
    load_pair_rows(dst, map, bar, kmajor, f0, k0, kTileF / 64);
  }
}

__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Arrives on the barrier at this offset in both CTAs once the MMAs so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Whether `ok` holds in all eight epilogue warps.
__device__ __forceinline__ bool epilogue_agrees(bool ok) {
  int all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred.aligned q, 5, 256, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(int(ok))
      : "memory");
  return all != 0;
}

// Tiles in groups of 8 token tiles that sweep the features together, so that
// the tiles in flight share their operands in L2.
__device__ __forceinline__ void wide_tile(int t, int f_tiles, int t_tiles, int* ft, int* tt) {
  constexpr int G = 8;
  const int group = t / (G * f_tiles);
  const int first = group * G;
  const int rows = min(G, t_tiles - first);
  const int r = t - first * f_tiles;
  *tt = first + r % rows;
  *ft = r / rows;
}

template <int PREC, bool kGated>
__global__ void __launch_bounds__(kWideThreads, 1) __cluster_dims__(2, 1, 1)
    linear_wide_kernel(const __grid_constant__ LinMaps maps,
                       const __grid_constant__ LinEpilogue e, int k, int bt, int f_tiles, int t_tiles) {
  using C = WideCfg<PREC>;
  constexpr int kOut = kGated ? kTileF / 2 : kTileF;  // outputs per CTA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* exchange = reinterpret_cast<float*>(smem + C::kStages * C::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStage + C::kExchange);
  uint64_t* empty = full + C::kStages;
  uint64_t* tmem_full = empty + C::kStages;        // [kWideBufs]
  uint64_t* tmem_empty = tmem_full + kWideBufs;    // [kWideBufs], the leader's are used
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + kWideBufs);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  const int pairs = gridDim.x / 2, first = blockIdx.x / 2;
  const int k_tiles = (k + kBK - 1) / kBK;
  const int total = f_tiles * t_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kWideBufs; ++b) {
      mbar_init(&tmem_full[b], 1);
      mbar_init(&tmem_empty[b], 16);  // eight epilogue warps of each CTA
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_maps<PREC>(maps);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    // of both CTAs; fewer than 256 tokens fill part of a stage
    const uint32_t stage_bytes =
        2 * (kABytes * C::kAParts + uint32_t(bt / 2) * kBK * 2 * C::kBParts);
    const uint32_t leader_full = map_rank(smem_u32(full), 0);
    const bool leader = elect_one();
    Ring ring(1);  // of the stages' previous use; the first passes at once
    bool ready = false;
    for (int t = first; t < total && ok; t += pairs) {
      int ft, tt;
      wide_tile(t, f_tiles, t_tiles, &ft, &tt);
      const int f0 = (ft * 2 + rank) * kOut, t0 = tt * bt + rank * (bt / 2);
      for (int kt = 0; kt < k_tiles; ++kt) {
        const int s = ring.s;
        if (!ready) ok = lin_wait_warp(&empty[s], ring.phase);
        if (!ok) break;
        ring.next<C::kStages>();
        const bool peeked = lin_peek(&empty[ring.s], ring.phase);
        if (leader) {
          uint8_t* st = smem + s * C::kStage;
          if (rank == 0) mbar_expect_tx(&full[s], stage_bytes);
          const uint32_t bar = leader_full + uint32_t(s) * 8u;
          load_pair_features<kGated>(st, &maps.a_hi, bar, maps.a_kmajor, f0, e.feats, kt * kBK);
          if constexpr (C::kAParts == 2)
            load_pair_features<kGated>(st + kABytes, &maps.a_lo, bar, maps.a_kmajor, f0, e.feats,
                                       kt * kBK);
          uint8_t* sb = st + kABytes * C::kAParts;
          load_pair_rows(sb, &maps.b_hi, bar, maps.b_kmajor, t0, kt * kBK, bt / 128);
          if constexpr (C::kBParts == 2)
            load_pair_rows(sb + C::kBBytes, &maps.b_lo, bar, maps.b_kmajor, t0, kt * kBK, bt / 128);
        }
        ready = __all_sync(0xffffffffu, peeked);
      }
    }
    // every stage's last use has been signalled before this CTA leaves
    for (int i = 0; i < C::kStages && ok; ++i, ring.next<C::kStages>())
      ok = lin_wait_warp(&empty[ring.s], ring.phase);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = lin_idesc(256, bt, !maps.a_kmajor, !maps.b_kmajor);
      const LinDesc da(smem_u32(smem), maps.a_kmajor);
      const LinDesc db(smem_u32(smem) + kABytes * C::kAParts, maps.b_kmajor);
      const bool leader = elect_one();
      Ring ring(0);
      bool ready = false;
      int j = 0;
      for (int t = first; t < total && ok; t += pairs, ++j) {
        const int b = j % kWideBufs;
        if (j >= kWideBufs) ok = lin_wait_warp(&tmem_empty[b], (j / kWideBufs - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(b * kWideT);
        for (int kt = 0; kt < k_tiles; ++kt) {
          if (!ready) ok = lin_wait_warp(&full[ring.s], ring.phase);
          if (!ok) break;
          const int s = ring.s;
          ring.next<C::kStages>();
          // looked at before this stage's MMAs go out, read after them
          const bool peeked = lin_peek(&full[ring.s], ring.phase);
          const uint32_t off = uint32_t(s) * (C::kStage >> 4);
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < kBK / 16; ++ks) {
              const uint64_t dah = da.at(off, ks), dbh = db.at(off, ks);
              umma_pair(d, dah, dbh, idesc, (kt > 0 || ks > 0) ? 1u : 0u);
              if constexpr (PREC == 3)
                umma_pair(d, da.at(off + (kABytes >> 4), ks), dbh, idesc, 1u);
              if constexpr (PREC >= 2)
                umma_pair(d, dah, db.at(off + (C::kBBytes >> 4), ks), idesc, 1u);
            }
            commit_pair(&empty[s]);
          }
          ready = __all_sync(0xffffffffu, peeked);
        }
        if (!ok) break;
        if (leader) commit_pair(&tmem_full[b]);
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp & 3;  // lanes 32 quarter .. + 31
    const int odd = warp >= 6;     // warps 2-5 take the even 32-token runs, 6-9 the odd ones
    const int l = quarter * 32 + lane;
    const int half = quarter >> 1;  // SwiGLU: gate (0) or up (1) rows
    const int pair = (quarter & 1) + 2 * odd;  // of warps with the same features and tokens
    const uint32_t empty_at = map_rank(smem_u32(tmem_empty), 0);
    int j = 0;
    for (int t = first; t < total; t += pairs, ++j) {
      int ft, tt;
      wide_tile(t, f_tiles, t_tiles, &ft, &tt);
      const int b = j % kWideBufs;
      ok = lin_wait(&tmem_full[b], (j / kWideBufs) & 1) &&
           *reinterpret_cast<volatile int*>(&g_linear_status) == 0;
      tc_fence_after();
      __syncwarp();
      // the eight warps go on, or give up, together: they wait for one another below
      ok = epilogue_agrees(ok);
      if (!ok) break;
      const int f0 = (ft * 2 + rank) * kOut, t0 = tt * bt;
      const uint32_t lanes = tmem + uint32_t(b * kWideT) + (uint32_t(quarter * 32) << 16);
      const int f = f0 + (kGated ? l % kOut : l);
      const int row = kGated ? f + half * e.feats : f;  // row of w
      const bool on = f < e.feats;
      const float bias = e.bias && on ? e.bias[row] : 0.f;
      int turn = 0;
#pragma unroll 1
      for (int col = odd * 32; col < bt && t0 + col < e.toks; col += 64, turn ^= 1) {
        float v[32];
        __syncwarp();
        tmem_ld32(lanes + col, v);
        if (e.bias) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += bias;
        }
        if (e.pre) store_pre(e, row, on, t0 + col, e.toks, v);
        if constexpr (!kGated) {
          finish_run<false, 32>(e, f, t0 + col, e.toks, v, v);
        } else {
          // warps q (gate) and q + 2 (up) hold the same features: the gate warp
          // finishes the first 16 tokens of the run, the up warp the others
          float* box = exchange + (pair * 2 + turn) * 1024;
          float* to = box + (1 - half) * 512;
          float* from = box + half * 512;
          float mine[16], other[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            mine[i] = half ? v[16 + i] : v[i];
            to[i * 32 + lane] = half ? v[i] : v[16 + i];
          }
          asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory");
#pragma unroll
          for (int i = 0; i < 16; ++i) other[i] = from[i * 32 + lane];
          if (half == 0)
            finish_run<true, 16>(e, f, t0 + col, e.toks, mine, other);
          else
            finish_run<true, 16>(e, f, t0 + col + 16, e.toks, other, mine);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_remote(empty_at + uint32_t(b) * 8u);
    }
  }
  if (!ok) {  // let issued copies land before the CTA exits
    const uint64_t t = globaltimer();
    while (globaltimer() - t < 1000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------- host side
// 3-D tiled bf16 map of an operand: K-major boxes {64 k, box_rows}, MN-major
// boxes {64 columns, 64 k}; 128-byte swizzle.
bool lin_map(CUtensorMap* map, const void* p, bool kmajor, int64_t rows, int64_t k, int64_t ld,
             int box_rows) {
  EncodeTiledFn encode = encode_fn();
  if (!encode) return false;
  const int64_t inner = kmajor ? k : rows, outer = kmajor ? rows : k;
  const cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), 1};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * 2 * cuuint64_t(outer)};
  const cuuint32_t box[3] = {64, cuuint32_t(kmajor ? box_rows : kBK), 1};
  const cuuint32_t elem_strides[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box,
                elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BT, int PREC, bool kGated>
int launch_split(const LinMaps& maps, const LinEpilogue& e, int k, int splits, int64_t f_tiles,
                 int64_t t_tiles, cudaStream_t stream) {
  using C = SplitCfg<BT, PREC>;
  static std::atomic<bool> configured[kMaxDevices];
  auto kernel = linear_split_kernel<BT, PREC, kGated>;
  const int st = raise_smem(kernel, C::kSmem, configured);
  if (st != MR_OK) return st;
  const int64_t grid = f_tiles * t_tiles * splits;
  if (grid > 0x7fffffff) return MR_ERR_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, maps, e, k, splits, int(f_tiles));
  if (err != cudaSuccess) {
    set_cuda_error(err);
    cudaGetLastError();
    return MR_ERR_LAUNCH;
  }
  return launch_status();
}

template <int PREC, bool kGated>
int launch_wide(const LinMaps& maps, const LinEpilogue& e, int k, int bt, int64_t f_tiles,
                int64_t t_tiles, cudaStream_t stream) {
  using C = WideCfg<PREC>;
  static std::atomic<bool> configured[kMaxDevices];
  auto kernel = linear_wide_kernel<PREC, kGated>;
  const int st = raise_smem(kernel, C::kSmem, configured);
  if (st != MR_OK) return st;
  if (f_tiles * t_tiles > 0x7fffffff) return MR_ERR_ARGUMENT;
  const int64_t pairs = sm_count() / 2;
  const int64_t grid = 2 * (f_tiles * t_tiles < pairs ? f_tiles * t_tiles : pairs);
  kernel<<<unsigned(grid), kWideThreads, C::kSmem, stream>>>(maps, e, k, bt, int(f_tiles),
                                                            int(t_tiles));
  return launch_status();
}

struct LinPlan {
  int bt, splits;
  bool wide;
};

// The tile and the divisor of k with the shortest modelled time, in ns at
// full clock, from launches of 1 to 2048 tokens over six shapes of 0.8 M to
// 136 M weights (bf16; the choice was within 3 % of the fastest in the mean):
//   stage   64 k of one tile: what its loads and MMAs take, whichever is slower
//           (one product: 165, 205, 225 for 32, 64, 128 tokens of one CTA, 245
//           to 285 for 128 to 256 of a pair; each further product its MMAs)
//   rounds  tiles over the SMs, two small tiles to an SM at 1.6 times a stage
//   bounds  operand bytes from L2 at 18 TB/s, the weights from HBM at 6.2 TB/s
//           or 42 GB/s per CTA
// plus a launch's and an epilogue's fixed time; k is divided only where all the
// parts run at once.  splits != 0 fixes the divisor.
LinPlan plan_linear(int64_t feats, int64_t rows_w, int out_per_cta, int64_t toks, int64_t k,
                    int precision, int b_kmajor, int splits) {
  const double sms = double(sm_count());
  const double k_tiles = std::ceil(double(k) / kBK);
  const double weights = 2.0 * double(rows_w) * double(k);
  const int a_parts = precision == 3 ? 2 : 1, b_parts = precision >= 2 ? 2 : 1;
  LinPlan best{128, splits ? splits : 1, false};
  double best_cost = -1.0;
  auto consider = [&](LinPlan plan, double cost) {
    if (best_cost < 0.0 || cost < best_cost) {
      best = plan;
      best_cost = cost;
    }
  };
  auto bounded = [&](double work, double l2_bytes, double ctas) {
    const double hbm = std::min(6200.0, 42.0 * ctas);
    return std::max(work, std::max(l2_bytes / 18000.0, weights / hbm));
  };
  for (int bt : {16, 32, 64, 128}) {
    if ((bt < 64 && (toks > bt || !b_kmajor)) || (bt == 64 && toks > 512) ||
        (bt > 16 && toks <= bt / 2 && (b_kmajor || bt > 64)))
      continue;
    static const double kStage[3][3] = {{165, 260, 340}, {205, 280, 385}, {225, 345, 525}};
    const double tiles = std::ceil(double(feats) / out_per_cta) * std::ceil(double(toks) / bt);
    const int together = (precision == 1 && bt <= 64) || (precision == 2 && bt <= 32) ? 2 : 1;
    for (int s : {1, 2, 4, 8}) {
      if (splits ? s != splits : s > 1 && k_tiles / s < 4) continue;
      const double n = tiles * s;
      const double per = n <= sms ? 1 : together;
      const double rounds = std::ceil(n / (sms * per));
      if (!splits && s > 1 && rounds > 1) break;
      const double steps = std::ceil(k_tiles / s);
      const double stage = kStage[bt <= 32 ? 0 : bt / 64][precision - 1] * (per == 2 ? 1.6 : 1.0);
      const double fixed =
          4400 + 10.0 * bt + (s > 1 ? 300 + 100.0 * s + 6.0 * bt : 0.0) + (per == 2 ? 1500 : 0);
      const double bytes = n * steps * kBK * 2.0 * (kTileF * a_parts + bt * b_parts);
      consider({bt, s, false},
               fixed + bounded(rounds * steps * stage, bytes, std::min(n, sms * per)));
    }
  }
  for (int bt : {256, 224, 192, 160, 128}) {
    if (splits > 1 || toks < 64 || (!b_kmajor && bt % 128)) continue;
    const double tiles = std::ceil(double(feats) / (2 * out_per_cta)) * std::ceil(double(toks) / bt);
    const double pairs = std::floor(sms / 2);
    const double rounds = std::ceil(tiles / pairs);
    const double stage = std::max(245.0 + 0.31 * (bt - 128), 279.0 * precision * bt / 256.0);
    const double bytes = tiles * k_tiles * kBK * 2.0 * (2 * kTileF * a_parts + bt * b_parts);
    consider({bt, 1, true}, 4500 + 6.0 * bt +
                                bounded(rounds * k_tiles * stage, bytes,
                                        std::min(2 * tiles, sms)));
  }
  return best;
}

template <int PREC, bool kGated>
int run_linear(LinMaps& maps, const LinEpilogue& e, const void* a_hi, const void* a_lo, int64_t lda,
               const void* b_hi, const void* b_lo, int64_t ldb, int64_t rows_a, int64_t k,
               int splits, cudaStream_t stream) {
  constexpr int kOut = kGated ? kTileF / 2 : kTileF;
  const int64_t f_tiles = (int64_t(e.feats) + kOut - 1) / kOut;
  const LinPlan p =
      plan_linear(e.feats, rows_a, kOut, e.toks, k, PREC, maps.b_kmajor, splits);
  const int t_box = p.wide ? p.bt / 2 : p.bt;
  const bool good =
      lin_map(&maps.a_hi, a_hi, maps.a_kmajor, rows_a, k, lda, kOut) &&
      lin_map(&maps.b_hi, b_hi, maps.b_kmajor, e.toks, k, ldb, t_box) &&
      (PREC < 3 || lin_map(&maps.a_lo, a_lo, maps.a_kmajor, rows_a, k, lda, kOut)) &&
      (PREC < 2 || lin_map(&maps.b_lo, b_lo, maps.b_kmajor, e.toks, k, ldb, t_box));
  if (!good) return MR_ERR_ALIGNMENT;
  if (p.wide)
    return launch_wide<PREC, kGated>(maps, e, int(k), p.bt,
                                     (int64_t(e.feats) + 2 * kOut - 1) / (2 * kOut),
                                     (int64_t(e.toks) + p.bt - 1) / p.bt, stream);
  const int64_t t_tiles = (int64_t(e.toks) + p.bt - 1) / p.bt;
  switch (p.bt) {
    case 16: return launch_split<16, PREC, kGated>(maps, e, int(k), p.splits, f_tiles, t_tiles, stream);
    case 32: return launch_split<32, PREC, kGated>(maps, e, int(k), p.splits, f_tiles, t_tiles, stream);
    case 64: return launch_split<64, PREC, kGated>(maps, e, int(k), p.splits, f_tiles, t_tiles, stream);
    default: return launch_split<128, PREC, kGated>(maps, e, int(k), p.splits, f_tiles, t_tiles, stream);
  }
}

}  // namespace

int linear_status(int reset) {
  int v = 0;
  const cudaError_t e = cudaMemcpyFromSymbol(&v, g_linear_status, sizeof(int));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return MR_ERR_LAUNCH;
  }
  if (reset && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mr

using namespace mr;

extern "C" int mr_linear(const mr_linear_operand* x, const mr_linear_operand* w, int64_t toks,
                         int64_t feats, int64_t k, int act, const float* bias,
                         const void* residual, int residual_dtype, int64_t ldr, void* out,
                         int out_dtype, uint16_t* out_lo, float* out_t32, int64_t ldo, float* pre,
                         int64_t ldp, int splits, void* stream) {
  if (!x || !w || !x->hi || !w->hi || !out || toks <= 0 || feats <= 0 || k <= 0)
    return MR_ERR_ARGUMENT;
  const int64_t most = 0x7fffff00;  // tile origins stay 32-bit
  if (toks > most || feats > most / 2 || k > most || act < MR_ACT_NONE || act > MR_ACT_SWIGLU)
    return MR_ERR_ARGUMENT;
  if (splits != 0 && splits != 1 && splits != 2 && splits != 4 && splits != 8)
    return MR_ERR_ARGUMENT;
  const bool gated = act == MR_ACT_SWIGLU;
  if ((gated && !w->kmajor) || (w->lo && !x->lo)) return MR_ERR_ARGUMENT;
  if ((out_dtype != MR_F32 && out_dtype != MR_BF16) || (out_lo && out_dtype != MR_BF16) ||
      (residual && residual_dtype != MR_F32 && residual_dtype != MR_BF16))
    return MR_ERR_ARGUMENT;
  const int64_t rows_w = gated ? 2 * feats : feats;
  if ((x->kmajor ? x->ld < k : x->ld < toks) || (w->kmajor ? w->ld < k : w->ld < rows_w) ||
      ldo < feats || (residual && ldr < feats) || (pre && ldp < rows_w))
    return MR_ERR_ARGUMENT;
  if (!aligned16(x->hi) || !aligned16(x->lo) || !aligned16(w->hi) || !aligned16(w->lo) ||
      x->ld % 8 || w->ld % 8)
    return MR_ERR_ALIGNMENT;
  LinMaps maps;
  memset(&maps, 0, sizeof(maps));
  maps.a_kmajor = w->kmajor != 0;
  maps.b_kmajor = x->kmajor != 0;
  LinEpilogue e;
  e.bias = bias;
  e.residual = residual;
  e.out = out;
  e.lo = out_lo;
  e.t32 = out_t32;
  e.pre = pre;
  e.ldr = ldr;
  e.ldo = ldo;
  e.ldp = ldp;
  e.residual_dtype = residual_dtype;
  e.out_dtype = out_dtype;
  e.act = act;
  e.feats = int(feats);
  e.toks = int(toks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define MR_LINEAR(PREC)                                                                        \
  (gated ? run_linear<PREC, true>(maps, e, w->hi, w->lo, w->ld, x->hi, x->lo, x->ld, rows_w, k, \
                                  splits, st)                                                  \
         : run_linear<PREC, false>(maps, e, w->hi, w->lo, w->ld, x->hi, x->lo, x->ld, rows_w, k, \
                                   splits, st))
  if (w->lo) return MR_LINEAR(3);
  if (x->lo) return MR_LINEAR(2);
  return MR_LINEAR(1);
#undef MR_LINEAR
}
