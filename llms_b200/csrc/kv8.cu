// 8-bit KV cache: tokens in (append) and out again (expand).
//
// Block j of a (row, head) holds tokens 64 j .. 64 j + 63.  Over the tokens
// that are there, with a = max |x|:
//     s = fl32(a / 127),   q = round-half-even(x / s),   x' = q s.
// The rounding decides on the exact quotient, not on a rounded one: with
// t = round(x fl(1/s)), which is off by at most one, the remainder x - t s is
// exact in one fma and is compared with s / 2.  So the stored bits are a
// function of the tokens alone.  a == 0 gives s = 0, q = 0; an infinity or NaN
// among the tokens gives a scale that is not finite and q = 0, so that every
// value of the block reads as NaN.
//
// The scale of an open block moves as it fills.  Rescaling 8-bit values would
// round a token again each time, so the tokens of the block that the last
// append ended in are also kept as they came (the tail, 64 rows), and when the
// scale moves the block is quantised again from them: token by token gives the
// same bits as all at once, and writing a token again gives what writing it
// once gives.
//
// append: one CTA per (block, head, row) and K / V.  A CTA keeps its block (64
// tokens) in registers between the maximum and the rounding, so each token is
// read once.  Single tokens read the block's earlier tokens (at most 63 rows
// from the tail) and write one row of 8 bits while the scale stands.
// expand: 16 values per thread.
// Measured (B200, bf16, KV 8, D 128): 4096 tokens of one row in 9.3 us (25 MB moved,
// 2.7 TB/s; 8 MB of it stay in L2) and out in 7.0 us (3.6 TB/s), 4 x 1537 in 13.5 and
// 9.2; 3.8 us would be the copy rate.  Most of the append is integer instructions (the
// maximum, the packing, the test for a border: issue 66 %, special-function pipe 5 %) and
// its CTAs' waits for load, maximum and store in turn; the expansion has two loads a
// thread in flight and a division for each.
#include "kv8.cuh"

namespace b200mm {

namespace {

// 64 values per thread at D = 128, 16-bit: with 256 threads a third of the work was what each does once per block.
constexpr int kThreads = 128;

struct AppendArgs {
  b200mm_kv8 c;
  const void* src[2];
  int64_t sb[2], sh[2], st[2];
  int64_t T;
  Kv8Pos pos;
  bool late;  // the next kernel starts when the one before is done (see kv8_decode)
};

// The largest |x| of a 16-byte chunk and `mx` as bits that order like the values, NaN above
// infinity (two 16-bit halves at once).
template <typename T> __device__ __forceinline__ uint32_t max_bits(const uint4& v, uint32_t mx) {
  const uint32_t m = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  const uint32_t a = v.x & m, b = v.y & m, c = v.z & m, d = v.w & m;
  if constexpr (sizeof(T) == 2) return __vmaxu2(__vmaxu2(__vmaxu2(a, b), __vmaxu2(c, d)), mx);
  return max(max(max(a, b), max(c, d)), mx);
}
template <typename T> __device__ __forceinline__ uint32_t to_f32_bits(uint32_t mx) {  // of the larger half
  if constexpr (sizeof(T) == 4) return mx;
  const unsigned short h = (unsigned short)max(mx & 0xffffu, mx >> 16);
  return __float_as_uint(to_f<T>(*reinterpret_cast<const T*>(&h)));
}

// round-half-even(x / s) for |x| <= 127 s (1 + 2^-24), s >= 2^-125, inv = fl(1 / s), half =
// s / 2, in the low byte (two's complement).  Adding 1.5 2^23 rounds to a whole number in
// the low bits; `border`: the remainder reaches half a step, so settle() has the last word.
__device__ __forceinline__ uint32_t quantize(float x, float s, float inv, float half, bool& border) {
  const float y = fmaf(x, inv, 12582912.f);
  const float d = fmaf(-(y - 12582912.f), s, x);  // exact
  border |= fabsf(d) >= half;
  return __float_as_uint(y);
}
__device__ __forceinline__ uint32_t settle(float x, uint32_t t, float s, float half) {
  const float d = fmaf(-(__uint_as_float(t) - 12582912.f), s, x);
  if (fabsf(d) > half || (fabsf(d) == half && (t & 1))) t += d > 0.f ? 1 : -1;
  return t;
}

// The same for a scale below 2^-125, whose reciprocal may overflow.  In units of
// the smallest subnormal x and s are whole numbers (s is its own bits), s < 2^24 and
// |x| < 2^31: the quotient by division of whole numbers.
__device__ uint32_t quantize_tiny(float x, float s) {
  const uint32_t n = (uint32_t)(fabsf(x) * 0x1p+100f * 0x1p+49f), d = __float_as_uint(s);
  uint32_t t = n / d;
  const uint32_t r2 = 2 * (n - t * d);
  if (r2 > d || (r2 == d && (t & 1))) ++t;
  return (x < 0.f ? 0u - t : t) & 255;
}

// Quantise block `blk` of one (row, head): rows [0, r0) come from the tail,
// rows [r0, r1) from `src` (row r0's address), the rest is not there.
template <typename T, int NC>
__device__ void do_block(const T* src, int64_t src_st, T* tail, int8_t* qdst, float* sdst, int D, int r0, int r1,
                         bool write_tail, uint32_t* red) {
  constexpr int V = 16 / sizeof(T);  // elements per 16-byte chunk
  const int cpr = D / V;             // chunks per row
  const int total = r1 * cpr;
  // chunk i of this thread: row, column
  const bool even = kThreads % cpr == 0;
  const int row0 = threadIdx.x / cpr, col0 = threadIdx.x - row0 * cpr, rstep = kThreads / cpr;
  auto place = [&](int i, int& row, int& c) {
    if (even) {
      row = row0 + i * rstep;
      c = col0;
    } else {
      row = (threadIdx.x + i * kThreads) / cpr;
      c = threadIdx.x + i * kThreads - row * cpr;
    }
  };
  uint4 x[NC];
  uint32_t mx = 0;
  const uint32_t s_old = __float_as_uint(*sdst);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x + i * kThreads < total) {
      int row, c;
      place(i, row, c);
      const T* p = row < r0 ? tail + (int64_t)row * D : src + (int64_t)(row - r0) * src_st;
      x[i] = *reinterpret_cast<const uint4*>(p + c * V);
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) mx = max_bits<T>(x[i], mx);
  mx = to_f32_bits<T>(mx);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
  __syncthreads();  // (also: every thread has read s_old)
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) mx = max(mx, red[w]);
  const float s = __fdiv_rn(__uint_as_float(mx), 127.f);
  const bool all_rows = __float_as_uint(s) != s_old;
  const float inv = __frcp_rn(s);
  // a finite scale, its half exact, or a tiny one; otherwise (0, or not finite) all bits are 0
  const bool plain = mx < 0x7f800000u && s >= 0x1p-125f, tiny = s > 0.f && s < 0x1p-125f;
  const float half = 0.5f * s;
  if (write_tail)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int row, c;
      place(i, row, c);
      if (row >= r0 && row < r1) *reinterpret_cast<uint4*>(tail + (int64_t)row * D + c * V) = x[i];
    }
  // every chunk's bits; earlier rows only where the scale moved
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    int row, c;
    place(i, row, c);
    const bool store = row < r1 && (row >= r0 || all_rows);
    if (!__any_sync(0xffffffffu, store)) continue;
    float f[V];
    Chunk<T>::unpack(x[i], f);
    uint32_t t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = 0;
    if (plain) {
      bool border = false;
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = quantize(f[e], s, inv, half, border);
      // with care, where the warp has a value on a border (a value of half the largest is on
      // one, 127 being odd: one chunk of 256 bf16 values in five)
      if (__any_sync(0xffffffffu, border)) {
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = settle(f[e], t[e], s, half);
      }
    } else if (tiny) {
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = quantize_tiny(f[e], s);
    }
    if (!store) continue;
    int8_t* dst = qdst + (int64_t)row * D + c * V;
    uint32_t o[V / 4];
#pragma unroll
    for (int w = 0; w < V / 4; ++w)
      o[w] = __byte_perm(__byte_perm(t[4 * w], t[4 * w + 1], 0x0040), __byte_perm(t[4 * w + 2], t[4 * w + 3], 0x0040), 0x5410);
    if constexpr (V == 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    else
      *reinterpret_cast<uint32_t*>(dst) = o[0];
  }
  if (threadIdx.x == 0) *sdst = s;
}

// (many CTAs per SM: each waits for its maximum between reading and writing)
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads, NC == 8 ? 7 : 1) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ uint32_t red[kThreads / 32];
  if (!a.late) pdl_trigger();
  pdl_wait();
  if (a.late) pdl_trigger();
  // heads next to each other, K before V: together they read whole rows of a projection's output
  const int heads = 2 * a.c.KV, hw = blockIdx.x % heads, which = hw / a.c.KV, h = hw - which * a.c.KV, b = blockIdx.y;
  const int64_t p0 = a.pos(b);
  if (p0 < 0 || p0 >= a.c.S) return;  // a row that is not there, or past the capacity
  const int64_t p1 = p0 + a.T < a.c.S ? p0 + a.T : a.c.S;
  const int64_t first = p0 / kKv8Block, last = (p1 - 1) / kKv8Block;
  const int D = a.c.D, r0 = (int)(p0 % kKv8Block);
  const T* src = static_cast<const T*>(a.src[which]) + (int64_t)b * a.sb[which] + (int64_t)h * a.sh[which];
  T* tail = static_cast<T*>(which ? a.c.vt : a.c.kt) + (int64_t)b * a.c.t_sb + (int64_t)h * a.c.t_sh;
  int8_t* q = (which ? a.c.vq : a.c.kq) + (int64_t)b * a.c.q_sb + (int64_t)h * a.c.q_sh;
  float* s = (which ? a.c.vs : a.c.ks) + (int64_t)b * a.c.s_sb + (int64_t)h * a.c.s_sh;
  auto run = [&](int64_t blk) {
    const int64_t t0 = blk * kKv8Block;
    const int lo = blk == first ? r0 : 0;
    const int hi = (int)(p1 - t0 < kKv8Block ? p1 - t0 : kKv8Block);
    do_block<T, NC>(src + (t0 + lo - p0) * a.st[which], a.st[which], tail, q + t0 * D, s + blk, D, lo, hi, blk == last,
                    red);
  };
  const int64_t blk = first + blockIdx.x / heads;
  if (blk > last) return;
  // a first block that reads the tail and a last block that writes it are one CTA's, in this order
  const bool both = r0 > 0 && last > first;
  if (both && blk == last) return;
  run(blk);
  if (both && blk == first) {
    __syncthreads();
    run(last);
  }
}

struct ExpandArgs {
  b200mm_kv8 c;
  void* dst[2];
  int64_t o_sb, o_sh, o_st;
  int64_t L;
};

// 16 values of one token per thread and step.
template <typename T>
__global__ void __launch_bounds__(kThreads) kv8_expand_kernel(const __grid_constant__ ExpandArgs a) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, which = blockIdx.y & 1, h = blockIdx.y >> 1;
  const unsigned cpr = a.c.D / 16, n = (unsigned)a.L * cpr;  // (at most 2^24 tokens of 16 chunks)
  const int8_t* q = (which ? a.c.vq : a.c.kq) + (int64_t)b * a.c.q_sb + (int64_t)h * a.c.q_sh;
  const float* s = (which ? a.c.vs : a.c.ks) + (int64_t)b * a.c.s_sb + (int64_t)h * a.c.s_sh;
  T* dst = static_cast<T*>(a.dst[which]) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  constexpr int U = 2;  // steps at once
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < n; i += U * step) {
    uint4 v[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned k = i + u * step;
      if (k < n) {
        v[u] = __ldcs(reinterpret_cast<const uint4*>(q + (int64_t)k * 16));
        sc[u] = s[k / cpr / kKv8Block];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned k = i + u * step;
      if (k >= n) break;
      const unsigned t = k / cpr, c = k - t * cpr;
      float f[16];
      Chunk<int8_t>::unpack(v[u], f);
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int w = 0; w < 16 / V; ++w) {
        T o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = from_f<T>(f[w * V + e] * sc[u]);
        *reinterpret_cast<uint4*>(dst + (int64_t)t * a.o_st + 16 * c + w * V) = *reinterpret_cast<const uint4*>(o);
      }
    }
  }
}

template <typename T>
int append_t(const AppendArgs& a, int B, cudaStream_t st) {
  // blocks that T tokens touch, wherever they start
  const int64_t nb = (a.T + kKv8Block - 2) / kKv8Block + 1;
  const int64_t cap = a.c.S / kKv8Block;
  const dim3 grid((unsigned)((nb < cap ? nb : cap) * 2 * a.c.KV), B);
  // 64 D elements, 16 bytes per thread and step
  const size_t steps = (size_t)kKv8Block * a.c.D * sizeof(T) / 16 / kThreads;
  const cudaError_t e = steps <= 8    ? launch_pdl(kv8_append_kernel<T, 8>, grid, dim3(kThreads), 0, st, a)
                        : steps <= 16 ? launch_pdl(kv8_append_kernel<T, 16>, grid, dim3(kThreads), 0, st, a)
                                      : launch_pdl(kv8_append_kernel<T, 32>, grid, dim3(kThreads), 0, st, a);
  return e == cudaSuccess ? B200MM_OK : B200MM_ERR_LAUNCH;
}

template <typename T>
int expand_t(const ExpandArgs& a, int B, cudaStream_t st) {
  const int64_t n = a.L * (a.c.D / 16);
  const int64_t want = (n + 2 * kThreads - 1) / (2 * kThreads);
  const dim3 grid((unsigned)(want < 4096 ? want : 4096), 2 * a.c.KV, B);
  return launch_pdl(kv8_expand_kernel<T>, grid, dim3(kThreads), 0, st, a) == cudaSuccess ? B200MM_OK
                                                                                       : B200MM_ERR_LAUNCH;
}

}  // namespace

int kv8_append(const b200mm_kv8& c, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void* v,
               int64_t v_sb, int64_t v_sh, int64_t v_st, int B, int64_t T, Kv8Pos pos, bool late, cudaStream_t st) {
  const AppendArgs a{c, {k, v}, {k_sb, v_sb}, {k_sh, v_sh}, {k_st, v_st}, T, pos, late};
  if (c.dtype == B200MM_BF16) return append_t<__nv_bfloat16>(a, B, st);
  if (c.dtype == B200MM_F16) return append_t<__half>(a, B, st);
  return append_t<float>(a, B, st);
}

int kv8_expand(const b200mm_kv8& c, void* k, void* v, int64_t o_sb, int64_t o_sh, int64_t o_st, int B, int64_t L,
               cudaStream_t st) {
  const ExpandArgs a{c, {k, v}, o_sb, o_sh, o_st, L};
  if (c.dtype == B200MM_BF16) return expand_t<__nv_bfloat16>(a, B, st);
  if (c.dtype == B200MM_F16) return expand_t<__half>(a, B, st);
  return expand_t<float>(a, B, st);
}

}  // namespace b200mm
