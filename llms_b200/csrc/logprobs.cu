// Log probabilities of given tokens, entropy and top alternatives of logit rows:
//   lse = log sum_i e^x_i,  logprob = x[token] - lse,  H = lse - sum_i p_i x_i,
//   top: the largest x_i in descending order, ties by ascending index.
//
// A row is read once, 16 bytes per lane and four loads at a time.  Each thread
// keeps, over its share of the row, the maximum m, l = sum e^(x - m) and
// e = sum e^(x - m) (x - m) in fp32 (e in units of log 2), rescaled once per four
// loads; then lse = m + log l and H = log l - e / l.  An element costs its
// widening, one multiply-add, the exponential, an addition and a multiply-add.
//
// Top alternatives: 128 groups of threads each know the largest value of their
// shares.  The k-th largest of these is a bound that at least k elements
// reach, and only threads whose own largest reaches it hold any: their shares
// are read again (about k of them, a few KB of L2), the elements that reach the
// bound are collected and ranked by counting.  No sort, and no second pass over the row.
// Where more elements reach the bound than are kept (a row whose k-th value is
// the -infinity of a masked vocabulary, or all logits the same), the ones
// above it are collected and the lowest indices among the equal ones follow in
// a scan that ends as soon as there are enough.  Rows that defeat this too
// (thousands above the bound in the shares of few threads) and rows with NaN are
// searched once per alternative.
//
// Measured (151,936 bf16 logits): 2048 rows 102 us (6.1 TB/s), 108 with one alternative;
// 64 rows 9.5 and, with 20, 15; one row 3.9 and, with 5, 8.8.  Many rows are bound by
// the exponentials and the stream together (special-function pipe 65 %), few by the
// latency of one pass, the meeting of the CTAs and the alternatives' five steps.
//
// A cluster of up to 16 CTAs shares a row when there are few rows; sums and
// alternatives meet in the first CTA through distributed shared memory, so a
// call is one launch without a workspace.
#include "logprobs.cuh"

namespace b200mm {

namespace {

constexpr int kGroups = 128;              // groups of neighbouring threads
constexpr int kCand = 2048;               // elements collected at once
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kFar = -1000.f;           // 2^-1000 = 0: stands for -infinity where 0 * x has to be 0
static_assert(kLogprobsMaxTop <= kGroups, "the bound is one of the groups' largest values");

// Larger key: larger value (NaN above all, -0 and 0 the same), then smaller index.  0: none.
__device__ __forceinline__ uint32_t value_key(float x) {
  if (x != x) return 0xfffffffeu;  // (no key is all ones)
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t make_key(float x, uint32_t i) { return ((uint64_t)value_key(x) << 32) | (uint32_t)~i; }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? b ^ 0x80000000u : ~b);  // (NaN's key reads as a NaN)
}

struct Sums {
  float m, l, e;  // e: of (x - m) log2(e)
};
// max(d, kFar), NaN kept
__device__ __forceinline__ float near(float d) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(d), "f"(kFar));
  return y;
}
// Vec: 16 bytes of a row.  max4: the largest element.  floor4: elements no
// lower than kFloor, NaN kept: -infinity stands for a probability of 0 without 0 * infinity.
// That serves where the maximum lies within (kFloor / 2, kTop), far above kFloor and
// with room for the factor; other rows go element by element.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr uint32_t kLowest = 0xff800000u;  // -infinity
  static constexpr float kFloor = -1e38f, kTop = 1e38f;
  __device__ __forceinline__ static float max4(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ __forceinline__ static uint32_t floor1(uint32_t w) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(__uint_as_float(w)), "f"(kFloor));
    return __float_as_uint(y);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr uint32_t kLowest = 0xff80ff80u;
  static constexpr float kFloor = -1e38f, kTop = 1e38f;
  __device__ __forceinline__ static float max4(const uint4& v) {
    auto h = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
    return fmaxf(f.x, f.y);
  }
  __device__ __forceinline__ static uint32_t floor1(uint32_t w) {
    const __nv_bfloat162 y = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(kFloor));
    return *reinterpret_cast<const uint32_t*>(&y);
  }
};
template <> struct Vec<__half> {
  static constexpr uint32_t kLowest = 0xfc00fc00u;
  static constexpr float kFloor = -65504.f, kTop = 1e38f;
  __device__ __forceinline__ static float max4(const uint4& v) {
    auto h = [](const uint32_t& w) { return *reinterpret_cast<const __half2*>(&w); };
    const float2 f = __half22float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
    return fmaxf(f.x, f.y);
  }
  __device__ __forceinline__ static uint32_t floor1(uint32_t w) {
    const __half2 y = __hmax2_nan(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(kFloor));
    return *reinterpret_cast<const uint32_t*>(&y);
  }
};
template <typename T>
__device__ __forceinline__ uint4 floor4(const uint4& v) {
  return make_uint4(Vec<T>::floor1(v.x), Vec<T>::floor1(v.y), Vec<T>::floor1(v.z), Vec<T>::floor1(v.w));
}

// The maximum m's part in the exponents, in units of log 2: an element's is
// x log2(e) - base(m), with base(m) = m log2(e) rounded once, or (other rows, see Vec)
// (x - m) log2(e), where a product could overflow.  Nothing but the base enters the
// results, so its rounding does not: 2^-24 of a logit of 20,000 would be 1e-3.
template <typename T>
__device__ __forceinline__ bool plain_max(float m) { return m > Vec<T>::kFloor / 2 && m < Vec<T>::kTop; }
__device__ __forceinline__ float base_of(float m) { return __fmul_rn(m, kLog2e); }  // (never fused into what uses it)
template <typename T>
__device__ __forceinline__ float exponent(float x, float m) {
  return plain_max<T>(m) ? fmaf(x, kLog2e, -base_of(m)) : (x - (m == -INFINITY ? 0.f : m)) * kLog2e;
}
// `s` with its maximum raised to at least `m`
template <typename T>
__device__ __forceinline__ void raise(Sums& s, float m) {
  const float mn = fmaxf(s.m, m);
  // from base to base (a maximum that is not plain beside one that is differs by far more than kFar)
  const float d = fmaxf(plain_max<T>(mn) ? base_of(s.m) - base_of(mn) : exponent<T>(s.m, mn), kFar), f = ex2(d);
  s.e = (s.e + s.l * d) * f;
  s.l *= f;
  s.m = mn;
}
template <typename T>
__device__ __forceinline__ void add(Sums& s, float x) {
  const float d = near(exponent<T>(x, s.m)), p = ex2(d);
  s.l += p;
  s.e = fmaf(p, d, s.e);
}
// the 32 lanes' sums as one, on every lane
template <typename T>
__device__ __forceinline__ Sums join(Sums s) {
  raise<T>(s, key_value((uint64_t)__reduce_max_sync(0xffffffffu, value_key(s.m)) << 32));
  return Sums{s.m, warp_sum(s.l), warp_sum(s.e)};
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

template <typename T, int kThreads, int kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) logprobs_kernel(const LogprobsArgs a, const int C) {
  constexpr int kWarps = kThreads / 32;
  constexpr int kPer = kThreads / kGroups;
  constexpr int VEC = 16 / sizeof(T);
  constexpr int U = 4;  // loads in flight per thread
  __shared__ uint64_t cand[kCand];
  __shared__ uint64_t list[kLogprobsMaxTop];
  __shared__ uint64_t lists[kMaxCluster][kLogprobsMaxTop];  // of every CTA (first CTA only)
  __shared__ float4 all[kMaxCluster];  // the CTAs' m, l, e
  __shared__ Sums wsum[kWarps];
  __shared__ uint64_t wkey[kWarps];
  __shared__ int wcount[kWarps];
  __shared__ __align__(16) float gbest[kGroups];
  __shared__ unsigned short holders[kThreads];  // threads whose largest value reaches the bound
  __shared__ float bound;
  __shared__ int ncand, nholders;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = C > 1 ? (int)cluster_rank() : 0;
  const int64_t row = blockIdx.x / C;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const int V = a.V, top = a.top;
  if (C > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();

  // the row: `head` elements up to a 16-byte boundary, nv vectors, a tail; the
  // first CTA's first threads take the single elements
  const int off = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int head = off ? min(V, VEC - off) : 0;
  const int nv = (V - head) / VEC;
  const int tail0 = head + nv * VEC;
  const T* xv = x + head;
  const int step = C * kThreads;
  const int v0 = rank * kThreads + tid;
  auto vec_at = [&](int v) { return *reinterpret_cast<const uint4*>(xv + (int64_t)v * VEC); };
  auto unpack = [&](const uint4& v, float* f) { Chunk<T>::unpack(v, f); };
  const bool has_head = rank == 0 && tid < head, has_tail = rank == 0 && tid < V - tail0;

  // ---- the stream ----
  Sums s{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  for (int v = v0; v < nv; v += U * step) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
      if (v + u * step < nv) w[u] = vec_at(v + u * step);
    }
    float mx = Vec<T>::max4(w[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) mx = fmaxf(mx, Vec<T>::max4(w[u]));
    best = fmaxf(best, mx);
    raise<T>(s, mx);
    if (plain_max<T>(s.m)) {
      const float ref = base_of(s.m);
      float l[2] = {s.l, 0.f}, e[2] = {s.e, 0.f};  // (two sums: a chain each)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VEC];
        unpack(floor4<T>(w[u]), f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = fmaf(f[i], kLog2e, -ref), p = ex2(d);
          l[i & 1] += p;
          e[i & 1] = fmaf(p, d, e[i & 1]);
        }
      }
      s.l = l[0] + l[1];
      s.e = e[0] + e[1];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VEC];
        unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) add<T>(s, f[i]);
      }
    }
  }
  auto single = [&](int i) {
    const float f = to_f<T>(x[i]);
    best = fmaxf(best, f);
    raise<T>(s, f);
    add<T>(s, f);
  };
  if (has_head) single(tid);
  if (has_tail) single(tail0 + tid);

  Sums t = join<T>(s);
  if (lane == 0) wsum[warp] = t;
  if (top > 0) {
    float g = best;
#pragma unroll
    for (int o = 1; o < kPer; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % kPer == 0) gbest[tid / kPer] = g;
    if (tid < kLogprobsMaxTop) list[tid] = 0;
    if (tid == 0) ncand = nholders = 0;
  }
  __syncthreads();
  const Sums none{-INFINITY, 0.f, 0.f};
  t = join<T>(lane < kWarps ? wsum[lane] : none);

  // ---- the CTA's alternatives, in order, to list[0 .. top) ----
  if (top > 0) {
    if (top > 1) {  // a group is ranked by its kPer threads, a share of the others each
      const int grp = tid / kPer, q = tid % kPer;
      const float g = gbest[grp];
      int above = 0, before = 0;  // larger ones; equal ones with a smaller number
#pragma unroll
      for (int i = 0; i < kGroups / kPer / 4; ++i) {
        const int at = q * (kGroups / kPer) + 4 * i;
        const float4 o = *reinterpret_cast<const float4*>(&gbest[at]);
        above += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
        before += (o.x == g && at < grp) + (o.y == g && at + 1 < grp) + (o.z == g && at + 2 < grp) + (o.w == g && at + 3 < grp);
      }
#pragma unroll
      for (int o = 1; o < kPer; o <<= 1) {
        above += __shfl_xor_sync(0xffffffffu, above, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
      }
      if (q == 0 && above + before == top - 1) bound = g;  // the top-th largest
      __syncthreads();
    }
    const float tau = top > 1 ? bound : t.m;
    if (best >= tau) holders[atomicAdd(&nholders, 1)] = (unsigned short)tid;
    __syncthreads();
    // their elements that reach the bound (`strict`: that lie above it); a
    // holder's vectors go to 2^lg lanes
    const int iters = max(0, (nv - rank * kThreads + step - 1) / step);  // of the CTA's first thread
    const int lg = iters > 16 ? 5 : iters > 8 ? 4 : iters > 4 ? 3 : iters > 2 ? 2 : 1;
    auto collect = [&](bool strict) {
      auto offer = [&](float f, int i) {
        if (strict ? f > tau : f >= tau) {
          const int at = atomicAdd(&ncand, 1);
          if (at < kCand) cand[at] = make_key(f, (uint32_t)i);
        }
      };
      for (int h = tid >> lg; h < nholders; h += kThreads >> lg) {
        const int first = rank * kThreads + holders[h];
#pragma unroll 2
        for (int it = tid & ((1 << lg) - 1); it < iters; it += 1 << lg) {
          const int v = first + it * step;
          if (v < nv) {
            const uint4 w = vec_at(v);
            if (Vec<T>::max4(w) >= tau) {
              float f[VEC];
              unpack(w, f);
#pragma unroll
              for (int j = 0; j < VEC; ++j) offer(f[j], head + v * VEC + j);
            }
          }
        }
      }
      if (has_head) offer(to_f<T>(x[tid]), tid);
      if (has_tail) offer(to_f<T>(x[tail0 + tid]), tail0 + tid);
    };
    auto rank_candidates = [&]() {
      const int n = ncand;
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t k = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > k;
        if (r < top) list[r] = k;
      }
    };
    bool search = !(t.l == t.l);  // NaN in the CTA's share (its values are not in the groups' largest)
    if (!search) {
      collect(false);
      __syncthreads();
      if (ncand <= kCand) {
        rank_candidates();
      } else {
        __syncthreads();  // every thread has read ncand
        if (tid == 0) ncand = 0;
        __syncthreads();
        collect(true);
        __syncthreads();
        search = ncand > kCand;
        if (!search) {
          rank_candidates();
          // equal ones, in the order of their indices
          int have = ncand;
          auto equal = [&](int c, uint32_t i0, uint32_t mask) {  // c of them here, at i0 + the bits of mask
            int inc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int y = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += y;
            }
            if (lane == 31) wcount[warp] = inc;
            __syncthreads();
            int before = 0, total = 0;
            for (int w = 0; w < kWarps; ++w) {
              if (w < warp) before += wcount[w];
              total += wcount[w];
            }
            int at = have + before + inc - c;
            while (mask && at < top) {
              list[at++] = make_key(tau, i0 + __ffs(mask) - 1);
              mask &= mask - 1;
            }
            have += total;
            __syncthreads();
          };
          {
            const bool e = has_head && to_f<T>(x[tid]) == tau;
            equal(e, tid, e);
          }
          for (int v = rank * kThreads; v < nv && have < top; v += step) {
            uint32_t mask = 0;
            if (v + tid < nv) {
              float f[VEC];
              unpack(vec_at(v + tid), f);
#pragma unroll
              for (int j = 0; j < VEC; ++j) mask |= (f[j] == tau ? 1u : 0u) << j;
            }
            equal(__popc(mask), (uint32_t)(head + (v + tid) * VEC), mask);
          }
          if (have < top) {
            const bool e = has_tail && to_f<T>(x[tail0 + tid]) == tau;
            equal(e, tail0 + tid, e);
          }
        }
      }
    }
    if (search) {  // the largest key below the last one found, `top` times
      uint64_t last = ~0ull;
      for (int k = 0; k < top; ++k) {
        uint64_t mine = 0;
        auto offer = [&](float f, int i) {
          const uint64_t key = make_key(f, (uint32_t)i);
          if (key < last && key > mine) mine = key;
        };
        for (int v = v0; v < nv; v += step) {
          float f[VEC];
          unpack(vec_at(v), f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) offer(f[j], head + v * VEC + j);
        }
        if (has_head) offer(to_f<T>(x[tid]), tid);
        if (has_tail) offer(to_f<T>(x[tail0 + tid]), tail0 + tid);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t y = __shfl_xor_sync(0xffffffffu, mine, o);
          mine = y > mine ? y : mine;
        }
        if (lane == 0) wkey[warp] = mine;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) mine = wkey[w] > mine ? wkey[w] : mine;
        if (tid == 0) list[k] = mine;
        last = mine;
        __syncthreads();
        if (last == 0) break;  // the CTA's share has no more
      }
    }
    __syncthreads();
  }

  // ---- the CTAs of a row meet in the first ----
  if (C > 1) {
    cluster_wait();
    if (tid < top) st_cluster_u64(map_to_rank(&lists[rank][tid], 0), list[tid]);
    if (tid == 0) st_cluster_f4(map_to_rank(&all[rank], 0), t.m, t.l, t.e, 0.f);
    cluster_sync();
    if (rank != 0) return;
    t = join<T>(lane < C ? Sums{all[lane].x, all[lane].y, all[lane].z} : none);
    for (int i = tid; i < C * top; i += kThreads) {
      const uint64_t k = lists[i / top][i % top];
      if (k == 0) continue;
      // keys are distinct and each list is in order: its own rank is the place
      // in its list plus what is larger in the others
      int r = i % top;
      for (int c = 0; c < C && r < top; ++c) {
        if (c == i / top) continue;
        for (int j = 0; j < top && lists[c][j] > k; ++j) ++r;
      }
      if (r < top) list[r] = k;
    }
    __syncthreads();
  }

  // nothing but -infinity: no distribution
  const float log_l = t.m == -INFINITY ? __int_as_float(0x7fc00000) : log2f(t.l);
  auto logprob = [&](float f) {  // (far out, where the factor could overflow, the base's rounding is nothing)
    return fabsf(f) < 1e30f ? (exponent<T>(f, t.m) - log_l) * kLn2 : (f - t.m) - log_l * kLn2;
  };
  if (tid == 0) {
    const int64_t tok = a.tokens[row];
    a.logprob[row] = tok >= 0 && tok < V ? logprob(to_f<T>(x[tok])) : __int_as_float(0x7fc00000);
    a.entropy[row] = (log_l - t.e / t.l) * kLn2;
  }
  if (tid < top) {
    const uint64_t k = list[tid];
    a.top_ids[row * top + tid] = (int64_t)(~(uint32_t)k);
    a.top_logprobs[row * top + tid] = logprob(key_value(k));
  }
}

template <typename T, int kThreads, int kCtas>
int launch(const LogprobsArgs& a, cudaStream_t st) {
  auto kern = logprobs_kernel<T, kThreads, kCtas>;
  const int dev = current_device();
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64) return B200MM_ERR_DEVICE;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return B200MM_ERR_LAUNCH;
    configured[dev] = true;
  }
  // CTAs per row: as many as are resident at once, up to 16 (a cluster), while
  // each has at least one 16-byte load for every thread
  const int64_t want = (int64_t)kCtas * num_sms(dev);
  int c = 1;
  while (c < kMaxCluster && a.M * (2 * c) <= want && (int64_t)a.V >= (int64_t)2 * c * kThreads * (16 / (int)sizeof(T)))
    c *= 2;
  const dim3 grid((unsigned)(a.M * c));
  const cudaError_t e = c > 1 ? launch_pdl_cluster(kern, grid, dim3(kThreads), 0, st, c, a, c)
                              : launch_pdl(kern, grid, dim3(kThreads), 0, st, a, c);
  return e == cudaSuccess ? B200MM_OK : B200MM_ERR_LAUNCH;
}

// Small CTAs for many rows: while one of six is at its sums and alternatives
// the others stream.  Large ones for few: a row's threads then meet in fewer
// steps.  (151,936 bf16 logits, device time: 2048 rows 102 us as 6 x 256 threads
// per SM and 121 as 2 x 512, 256 rows 26 and 18.)
template <typename T>
int launch(const LogprobsArgs& a, cudaStream_t st) {
  return a.M >= 4 * (int64_t)num_sms(current_device()) ? launch<T, 256, 6>(a, st) : launch<T, 512, 2>(a, st);
}

}  // namespace

int logprobs_launch(const LogprobsArgs& a, int dtype, cudaStream_t st) {
  if (dtype == B200MM_BF16) return launch<__nv_bfloat16>(a, st);
  if (dtype == B200MM_F16) return launch<__half>(a, st);
  return launch<float>(a, st);
}

}  // namespace b200mm
