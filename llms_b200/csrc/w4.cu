// Projections with 4-bit weights and group scales:
//   y[m, n] = epilogue(sum_k x[m, k] (u[n, k] - 8) s[n, k / G]),  G = 32, 64 or 128.
//
// Up to 64 rows of x the weights (0.5 byte each) would stream at 13e12 a second
// on this GPU: one fp32 multiply-add per weight on the CUDA cores would already
// take longer, so the products run on mma.sync m16n8k16 from one row of x on, and
// what is left per weight is its way from four bits to sixteen:
//   * a warp owns 16 weight rows; lane l reads 16 bytes (32 weights) of rows
//     l / 4 and l / 4 + 8 as they lie in memory, a chunk of 128 columns per warp;
//   * the products of one instruction have to lie in one group, so for G = 64
//     and 32 the four lanes of a row exchange words (one round of shuffles, or
//     two: a 4 x 4 transpose).  The order of k inside a group is free: x is
//     staged in shared memory in the order that the lanes hold the weights;
//   * four bits under the exponent of 2^10 (fp16; 2^7 for bf16 in the cluster kernel)
//     are 1024 + u: one logic instruction per pair, one packed subtraction,
//     exact.  Pairs are the weights 4 apart in a 32-bit word;
//   * a group's products are summed in fp32 in accumulators of their own, which
//     its scale then joins to the row's: no product is rounded;
//   * before griddepcontrol.wait a CTA only asks for its first weights in L2.
// Up to 16 rows of x and 4096 columns, one persistent CTA per SM walks tiles of 16
// weight rows.  Its warps split K; each has the part of x that it needs in registers
// and fills a ring of its own with cp.async, several tiles ahead, so only the sums
// of a tile meet at a barrier.  With more columns x lies in shared memory, where up to 8
// rows of it fit beside the rings (stream_fits: 8 rows at 5120 columns, 5 at 8192, 3 at
// 12288).  Otherwise K is split over a cluster of CTAs with 128 weight rows each, and
// the sums meet in distributed shared memory (12288 x 4096 gate and up: one row 25 us
// there and 16 in the persistent kernel, 16 rows 50 and 28; 4096 x 12288: 3 rows 14.5
// us here, 4 to 8 rows 16.5 there; 4096 x 8192: 5 rows 12.4, 6 to 8 rows 12.3), as many
// rows of x a launch as shared memory takes (rows_per_launch), each launch reading
// all weights: 4096 x 12288 26.6 us at 32 rows, 52 at 64 in two launches.
// From kDenseRows on the weights are expanded to 16 bits (rounded once: the
// tcgen05 GEMM's operands are 16-bit) into the caller's workspace and the dense
// GEMM takes them.  12288 x 4096 gate and up: 114 us at 128 rows, where two launches
// of 64 take 165; 83 us at 64 rows, where this would take 127 (65 to 80 rows would
// still be 100 to 112 in two launches, but 4096 x 12288 69 to 84 instead of 66).
// Measured (weights rotated past L2, G = 128): 12288 x 4096 gate and up 16.6 us at one
// row (3.1 TB/s), 19.0 at 8, 28.8 at 16, 47 at 32; 6144 x 4096 6.4-6.9 us at one row,
// 10.7 at 16.  Not HBM bounds these but instructions and fetching them: issue slots
// half full, no pipe full, four warps per scheduler.  (From 17 rows on the dense
// projections with 16-bit weights are as fast, 45 us there, and at 64 rows faster, 50.)
#include "w4.cuh"

#include <type_traits>

#include "dense.cuh"

namespace b200mm {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16 * kWarps;  // weight rows per CTA (and matrix)
constexpr int kChunk = 128;         // columns per warp and step
constexpr int kMaxRows = 64;        // rows of x per launch
constexpr int kDenseRows = 65;      // from here on: expand and run the dense GEMM
constexpr size_t kFenceBytes = 16;  // of workspace that the memset between the two writes

struct W4Params {
  const void* x; int64_t ldx;
  const uint8_t* w[2]; int64_t ldw;
  const void* s[2]; int64_t lds;
  void* y; int64_t ldy;
  int M, N, K;
  int kslice;  // columns per cluster rank (multiple of kChunk)
};

template <typename T> struct Nib;
template <> struct Nib<__nv_bfloat16> {
  // weights i and i + 4 of a word -> (u - 8) pair
  __device__ __forceinline__ static uint32_t pair(uint32_t w, int i) {
    const uint32_t h = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&h), __float2bfloat162_rn(136.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ static void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Nib<__half> {
  __device__ __forceinline__ static uint32_t pair(uint32_t w, int i) {
    const uint32_t h = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1032.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ static void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    mma_h(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};

// 8 values of x in the order of a word's pairs: 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 pair_order(const uint4& v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// First column (inside a chunk) of the 8 weights that lane c of a row holds in
// word j after spread(): words j of the four lanes lie in one group.
template <int G>
__device__ __forceinline__ int word_col(int j, int c) {
  if (G == 128) return 32 * c + 8 * j;
  if (G == 64) return 64 * (j >> 1) + 32 * (c & 1) + 16 * (c >> 1) + 8 * (j & 1);
  return 32 * j + 8 * c;
}
template <int G>
__device__ __forceinline__ void spread(uint32_t (&w)[4], int c) {
  if constexpr (G <= 64) {  // the far half of the words with the lane two away
    const bool up = c & 2;
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[2], 2);
    const uint32_t r1 = __shfl_xor_sync(0xffffffffu, up ? w[1] : w[3], 2);
    if (up) {
      w[0] = r0;
      w[1] = r1;
    } else {
      w[2] = r0;
      w[3] = r1;
    }
  }
  if constexpr (G == 32) {  // and every other word with the neighbour
    const bool up = c & 1;
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[1], 1);
    const uint32_t r1 = __shfl_xor_sync(0xffffffffu, up ? w[2] : w[3], 1);
    if (up) {
      w[0] = r0;
      w[2] = r1;
    } else {
      w[1] = r0;
      w[3] = r1;
    }
  }
}

// ---------------------------------------------------------------------------
// persistent kernel: M <= 8 MT rows of x
// ---------------------------------------------------------------------------
constexpr int kStreamWarps = 16;    // at most
constexpr int kSlice = 2 * kChunk;  // columns per warp and step: 128 bytes of a row

// Ring slots per warp (2 KB of each matrix a slot).
__host__ __device__ constexpr int stream_depth(bool gate, bool xreg) { return (xreg ? 6 : 4) / (gate ? 2 : 1); }

// The eight weights of a word as four pairs, (0, 4), (1, 5), (2, 6), (3, 7).  fp16:
// under the exponent of 2^10 a low half is 1024 + u, a high half 1024 + 16 u, so
// one shift serves two logic instructions (bf16's 7 bits want one each).  The way is
// that of Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run" (2022).
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(bits));
  return v;
}
template <typename W>
__device__ __forceinline__ void nibbles(uint32_t w, uint32_t (&o)[4]) {
  if constexpr (std::is_same<W, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = Nib<W>::pair(w, i);
    return;
  }
  const __half2 low = __float2half2_rn(-1032.f), k = __float2half2_rn(0.0625f), high = __float2half2_rn(-72.f);
  uint32_t v[4] = {and_or(w, 0x000f000fu, 0x64006400u), and_or(w, 0x00f000f0u, 0x64006400u),
                   and_or(w >> 8, 0x000f000fu, 0x64006400u), and_or(w >> 8, 0x00f000f0u, 0x64006400u)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = *reinterpret_cast<const __half2*>(&v[i]);
    const __half2 q = i & 1 ? __hfma2(h, k, high) : __hadd2(h, low);
    o[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
}

// Eight bf16 values of x as fp16, times `up`, in the order of a word's pairs.
__device__ __forceinline__ uint4 scaled_pairs(const uint4& v, float up) {
  float f[8];
  Chunk<__nv_bfloat16>::unpack(v, f);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[i] * up, f[i + 4] * up);
    o[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// Magnitudes of bf16 values, as their bits, two at a time: the largest and the smallest ...
struct Spread {
  uint32_t most = 0, least = ~0u;
  __device__ __forceinline__ void take(const uint4& v) {
    const uint32_t m = 0x7fff7fffu, a = v.x & m, b = v.y & m, c = v.z & m, d = v.w & m;
    most = __vmaxu2(most, __vmaxu2(__vmaxu2(a, b), __vmaxu2(c, d)));
    least = __vminu2(least, __vminu2(__vminu2(a, b), __vminu2(c, d)));
  }
  __device__ __forceinline__ uint32_t largest() const { return max(most >> 16, most & 0xffffu); }
  __device__ __forceinline__ uint32_t smallest() const { return min(least >> 16, least & 0xffffu); }
};
// ... and bits 15 and 31 set in `lost` where one is not zero and below `least`.  (a + 0x7fff has
// bit 15 set from a = 1 on, a + 0x8000 - least from a = least on; no half carries into the next.)
__device__ __forceinline__ uint32_t below(const uint4& v, uint32_t least, uint32_t lost) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w}, m = 0x7fff7fffu, k = 0x80008000u - least * 0x00010001u;
#pragma unroll
  for (int i = 0; i < 4; ++i) lost |= ((w[i] & m) + m) & ~((w[i] & m) + k);
  return lost;
}
// fp16 with the largest below 2^15 holds 8 bits from 2^-17 on: exponents at most 31 apart
// (below the normal numbers, where steps no longer shrink, the last normal one's counts).
__device__ __forceinline__ uint32_t least_bits(uint32_t most) { return most < 33u << 7 ? 0u : ((most >> 7) - 31) << 7; }
__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }
// The power of two that brings `mx` into [2^14, 2^15), and its inverse (both normal).
__device__ __forceinline__ float x_up(float mx, float& down) {
  const int e = max(1, min(268 - (int)(__float_as_uint(mx) >> 23), 253));
  down = __uint_as_float((uint32_t)(254 - e) << 23);
  return __uint_as_float((uint32_t)e << 23);
}

template <typename T>
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const unsigned short h = (unsigned short)bits;
  return to_f<T>(*reinterpret_cast<const T*>(&h));
}

// Products are exact.  fp16 weights take fewer instructions to widen than bf16 ones
// (12288 x 4096 gate and up, one row: 16.1 us, 18.9 with bf16), so up to 8 bf16 rows
// of x become fp16 too, by a power of two per slice of K and row that brings the
// largest element into [2^14, 2^15) and that the sums are scaled back by.  Where one
// of a slice's elements would lose bits that way (its exponent lies more than 31
// below the largest) the products are in bf16; looking for one costs 0.4 us.  (9 to
// 16 rows 27.3 and 28.0 us, 6144 x 4096 10.2 and 9.6: bf16 there, without the factors'
// registers.)
// XREG: every warp has one slice of K, and its part of x stays in registers;
// otherwise all of x is staged in shared memory.
template <typename T, int MT, int G, bool GATE, bool XREG>
__global__ void __launch_bounds__(32 * kStreamWarps, 1) w4_stream_kernel(const __grid_constant__ W4Params p, const int meet_tiles) {
  const int meet = MT == 1 ? meet_tiles : 1;  // (16 rows: no room for more than one, nor registers to count them)
  constexpr bool HALF = std::is_same<T, __nv_bfloat16>::value && MT == 1;  // bf16 x as fp16 where that is exact
  constexpr int NM = GATE ? 2 : 1;
  constexpr int D = stream_depth(GATE, XREG);
  constexpr int GPC = kChunk / G;  // groups per chunk
  constexpr int WPG = 4 / GPC;     // words of a lane per group
  constexpr int SPL = G == 32 ? 2 : 1;  // scales of a slice per lane (4 lanes share a row)
  constexpr uint32_t MAT = 16 * 128;    // bytes of a slot, one matrix
  extern __shared__ __align__(128) unsigned char smem_raw[];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int M = p.M, N = p.N, K = p.K;
  const int nsl = (K + kSlice - 1) / kSlice;
  const int per = XREG ? 1 : (nsl + nw - 1) / nw;  // slices of a tile per warp: warp + nw i
  const int ntiles = (N + 15) / 16;
  const int mine_tiles = (ntiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // tiles blockIdx.x + i gridDim.x
  const int total = mine_tiles * per;

  unsigned char* ring = smem_raw + (size_t)warp * D * NM * MAT;
  const uint32_t ring_u = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  // the warps' sums of up to `meet` tiles, [tile][NM][warp][16][rp]: they meet that often
  float* red = reinterpret_cast<float*>(smem_raw + (size_t)nw * D * NM * MAT);
  const int rp = (M + 1) & ~1;
  const int red_n = NM * nw * 16 * rp;
  // Columns 2 q, 2 q + 1 of a row.  Sums are read a column at a time: where 16 rows of rp would meet
  // in two or four banks the pairs change places from row to row (16 rows of x: 33 -> 27 us).
  const int zs = rp == 16 ? 1 : 2, zm = rp == 16 ? 7 : rp == 8 ? 3 : 0;
  auto red_at = [&](int row, int q) { return row * rp + 2 * (q ^ ((row >> zs) & zm)); };
  const int xpitch = nsl * kSlice + 32;  // rows of x 64 bytes apart in the banks
  __half* xs = reinterpret_cast<__half*>(red + meet * red_n);             // [M][xpitch]
  float* xdown = reinterpret_cast<float*>(xs + (XREG ? 0 : (int64_t)M * xpitch));  // [nsl][8]: 1 / the slices' powers of two

  // ---- the load cursor: lane (r, c) takes 16 bytes at 16 c and 64 + 16 c of rows r and r + 8 ----
  int lt = blockIdx.x, li = 0, lit = 0;  // tile, slice number of the warp, item
  const int64_t tile_step = (int64_t)gridDim.x * 16;
  const uint8_t* wsrc[NM];
  const T* ssrc[NM];
#pragma unroll
  for (int mtx = 0; mtx < NM; ++mtx) {
    const int64_t row = (int64_t)blockIdx.x * 16 + r;
    wsrc[mtx] = p.w[mtx] + row * p.ldw + warp * (kSlice / 2) + 16 * c;
    ssrc[mtx] = static_cast<const T*>(p.s[mtx]) + row * p.lds + warp * (kSlice / G) + (G == 128 ? c & 1 : c);
  }
  // odd rows with their halves swapped: a fragment load takes 64 bytes of an even and of an odd row
  const uint32_t frag = ring_u + r * 128 + ((c ^ ((r & 1) << 2)) << 4);
  uint32_t sv[D][NM][2][SPL];  // scales as they are: converting them here would wait for them
  auto raw = [](const T* q) -> uint32_t { return *reinterpret_cast<const unsigned short*>(q); };
  auto load = [&](int u) {
    const int k0 = (warp + nw * li) * kSlice;
    if (lit < total && k0 < K) {
      const int row = lt * 16 + r;
      if (lt * 16 + 16 <= N && k0 + kSlice <= K) {
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* src = wsrc[mtx] + (h ? 8 * p.ldw : 0);
            const uint32_t dst = frag + (u * NM + mtx) * MAT + h * 1024;
            cp_async16(dst, src);
            cp_async16(dst ^ 64, src + 64);
#pragma unroll
            for (int q = 0; q < SPL; ++q) sv[u][mtx][h][q] = raw(ssrc[mtx] + (h ? 8 * p.lds : 0) + 4 * q);
          }
        }
      } else {
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* src = wsrc[mtx] + (h ? 8 * p.ldw : 0);
            const uint32_t dst = frag + (u * NM + mtx) * MAT + h * 1024;
            const bool in = row + 8 * h < N, a = in && k0 + 32 * c < K, b = in && k0 + kChunk + 32 * c < K;
            cp_async16(dst, a ? src : p.w[mtx], a);
            cp_async16(dst ^ 64, b ? src + 64 : p.w[mtx], b);
#pragma unroll
            for (int q = 0; q < SPL; ++q)
              sv[u][mtx][h][q] = in && k0 + ((G == 128 ? c & 1 : c) + 4 * q) * G < K
                                     ? raw(ssrc[mtx] + (h ? 8 * p.lds : 0) + 4 * q) : 0u;
          }
        }
      }
    }
    cp_commit();
    ++lit;
    const bool wrap = ++li == per;
    if (wrap) {
      li = 0;
      lt += gridDim.x;
    }
#pragma unroll
    for (int mtx = 0; mtx < NM; ++mtx) {  // (past the last item the addresses are not used)
      wsrc[mtx] += wrap ? tile_step * p.ldw - (int64_t)(per - 1) * nw * (kSlice / 2) : (int64_t)nw * (kSlice / 2);
      ssrc[mtx] += wrap ? tile_step * p.lds - (int64_t)(per - 1) * nw * (kSlice / G) : (int64_t)nw * (kSlice / G);
    }
  };
  {  // the first slices on their way to L2 (nothing is read before the wait)
    int t = blockIdx.x, i = 0;
#pragma unroll
    for (int u = 0; u < D; ++u) {
      const int kb = (warp + nw * i) * (kSlice / 2);
      if (lane < 16 && u < total && t * 16 + lane < N && kb < (K >> 1))
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx) prefetch_l2(p.w[mtx] + (int64_t)(t * 16 + lane) * p.ldw + kb);
      if (++i == per) {
        i = 0;
        t += gridDim.x;
      }
    }
  }
  pdl_trigger();
  pdl_wait();
#pragma unroll
  for (int u = 0; u < D; ++u) load(u);

  // ---- x, zero past M and K ----
  const T* x = static_cast<const T*>(p.x);
  uint4 xr[XREG ? 2 : 1][4][MT];  // of the warp's slice: chunk, word, n-tile
  float down[MT][2];              // of columns 8 t + 2 c, + 1
  bool wide = false;              // bf16 products (XREG: in this warp, otherwise in the CTA)
  if constexpr (XREG) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = r + 8 * t;
      Spread sp;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = warp * kSlice + hh * kChunk + word_col<G>(j, c);
          xr[hh][j][t] = make_uint4(0, 0, 0, 0);
          if (m < M && k < K) xr[hh][j][t] = *reinterpret_cast<const uint4*>(x + (int64_t)m * p.ldx + k);
          if constexpr (HALF) sp.take(xr[hh][j][t]);
        }
      float up = 1.f, dn = 1.f;
      if constexpr (HALF) {
        uint32_t most = sp.largest();
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (__any_sync(0xffffffffu, m < M && sp.smallest() < least_bits(most))) {  // a zero, or less
          uint32_t lost = 0;
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int j = 0; j < 4; ++j) lost = below(xr[hh][j][t], least_bits(most), lost);
          wide = __any_sync(0xffffffffu, lost & 0x80008000u);
        }
        if (!wide) up = x_up(bf16_value(most), dn);
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xr[hh][j][t] = HALF && !wide ? scaled_pairs(xr[hh][j][t], up) : pair_order(xr[hh][j][t]);
      down[t][0] = HALF ? __shfl_sync(0xffffffffu, dn, 8 * c) : 1.f;
      down[t][1] = HALF ? __shfl_sync(0xffffffffu, dn, 8 * c + 4) : 1.f;
    }
  } else {
    // a warp per row and slice; 8 columns from word_col(j, c) lie at 16-byte place 4 j + c of their chunk
    auto stage = [&]() {
      uint32_t lost = 0;
      for (int i = warp; i < M * nsl; i += nw) {
        const int m = i / nsl, sl = i - m * nsl;
        const int place = lane & 15, ch = 2 * sl + (lane >> 4);
        const int k = ch * kChunk + word_col<G>(place >> 2, place & 3);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < K) v = *reinterpret_cast<const uint4*>(x + (int64_t)m * p.ldx + k);
        float up = 1.f, dn = 1.f;
        if (HALF && !wide) {
          Spread sp;
          sp.take(v);
          const uint32_t most = __reduce_max_sync(0xffffffffu, sp.largest());
          lost = below(v, least_bits(most), lost);
          up = x_up(bf16_value(most), dn);
        }
        if (HALF && lane == 0) xdown[sl * 8 + m] = dn;
        *reinterpret_cast<uint4*>(xs + (int64_t)m * xpitch + ch * kChunk + place * 8) =
            HALF && !wide ? scaled_pairs(v, up) : pair_order(v);
      }
      return lost & 0x80008000u;
    };
    wide = __syncthreads_or(stage());
    if (wide) {
      stage();
      __syncthreads();
    }
  }

  float acc[NM][MT][4];
  auto clear = [&]() {
#pragma unroll
    for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mtx][t][e] = 0.f;
  };
  clear();
  auto products = [&](auto type, int u, int sl) {  // slot u with its part of x, weights widened to `type`
    using W = decltype(type);
    if constexpr (!XREG) {
      down[0][0] = HALF && 2 * c < M ? xdown[sl * 8 + 2 * c] : 1.f;
      down[0][1] = HALF && 2 * c + 1 < M ? xdown[sl * 8 + 2 * c + 1] : 1.f;
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      uint32_t wd[NM][2][4];
#pragma unroll
      for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(wd[mtx][h][0]), "=r"(wd[mtx][h][1]), "=r"(wd[mtx][h][2]), "=r"(wd[mtx][h][3])
                       : "r"((frag ^ (hh << 6)) + (u * NM + mtx) * MAT + h * 1024) : "memory");
          spread<G>(wd[mtx][h], c);
        }
#pragma unroll
      for (int g = 0; g < GPC; ++g) {
        float part[NM][MT][4];
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[mtx][t][e] = 0.f;
#pragma unroll
        for (int jj = 0; jj < WPG; ++jj) {
          const int j = g * WPG + jj;
          uint4 b[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if constexpr (XREG) {
              b[t] = xr[hh][j][t];
            } else {
              b[t] = make_uint4(0, 0, 0, 0);
              if (r + 8 * t < M)
                b[t] = *reinterpret_cast<const uint4*>(xs + (int64_t)(r + 8 * t) * xpitch + sl * kSlice + hh * kChunk + 32 * j + 8 * c);
            }
          }
#pragma unroll
          for (int mtx = 0; mtx < NM; ++mtx) {
            uint32_t lo[4], hi[4];
            nibbles<W>(wd[mtx][0][j], lo);
            nibbles<W>(wd[mtx][1][j], hi);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t a[4] = {lo[2 * q], hi[2 * q], lo[2 * q + 1], hi[2 * q + 1]};
#pragma unroll
              for (int t = 0; t < MT; ++t) Nib<W>::mma(part[mtx][t], a, q ? b[t].z : b[t].x, q ? b[t].w : b[t].y);
            }
          }
        }
        const int gi = hh * GPC + g;  // the group in the slice: held by lane gi % 4 of the row
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx) {
          const float s0 = scale_of<T>(__shfl_sync(0xffffffffu, sv[u][mtx][0][gi / 4], (lane & 28) + gi % 4));
          const float s1 = scale_of<T>(__shfl_sync(0xffffffffu, sv[u][mtx][1][gi / 4], (lane & 28) + gi % 4));
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = XREG || !HALF ? (e < 2 ? s0 : s1) : (e < 2 ? s0 : s1) * down[t][e & 1];
              acc[mtx][t][e] = fmaf(part[mtx][t][e], f, acc[mtx][t][e]);
            }
        }
      }
    }
  };
  int i = 0, done = 0;  // the item's number in its tile, tiles done
  for (int it0 = 0; it0 < total; it0 += D) {
#pragma unroll
    for (int u = 0; u < D; ++u) {
      if (it0 + u >= total) break;
      const int sl = warp + nw * i;
      cp_wait<D - 1>();
      __syncwarp();
      if (sl < nsl) {
        if (HALF && wide)
          products(__nv_bfloat16(), u, sl);
        else
          products(typename std::conditional<HALF, __half, T>::type(), u, sl);
      }
      __syncwarp();
      load(u);
      if (++i == per) {
        i = 0;
        float* mine = red + (done % meet) * red_n + warp * 16 * rp;
#pragma unroll
        for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (8 * t + 2 * c < M) {
                const float d0 = XREG ? down[t][0] : 1.f, d1 = XREG ? down[t][1] : 1.f;
                *reinterpret_cast<float2*>(mine + mtx * nw * 16 * rp + red_at(r + 8 * h, 4 * t + c)) =
                    make_float2(acc[mtx][t][2 * h] * d0, acc[mtx][t][2 * h + 1] * d1);
              }
        clear();
        if (++done % meet == 0 || done == mine_tiles) {
          const int first = (done - 1) / meet * meet;
          __syncthreads();
          for (int o = threadIdx.x; o < (done - first) * 16 * M; o += blockDim.x) {
            const int row = o % 16, m = MT == 1 ? o / 16 % M : o / 16, tl = MT == 1 ? o / (16 * M) : 0;
            const int n = ((int)blockIdx.x + (first + tl) * (int)gridDim.x) * 16 + row;
            const float* src = red + tl * red_n + red_at(row, m >> 1) + (m & 1);
            float v[NM];
#pragma unroll
            for (int mtx = 0; mtx < NM; ++mtx) {
              v[mtx] = 0.f;
#pragma unroll 4
              for (int w = 0; w < nw; ++w) v[mtx] += src[(mtx * nw + w) * 16 * rp];
            }
            if (n < N) static_cast<T*>(p.y)[(int64_t)m * p.ldy + n] = from_f<T>(GATE ? silu_mul(v[0], v[NM - 1]) : v[0]);
          }
          if (done < mine_tiles) __syncthreads();  // (before the next tiles' sums)
        }
      }
    }
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------
// cluster kernel
// ---------------------------------------------------------------------------
// MT: n-tiles of 8 rows of x; CS: CTAs of a cluster (K split).
template <typename T, int MT, int G, bool GATE, int CS>
__global__ void __launch_bounds__(kThreads) w4_kernel(const __grid_constant__ W4Params p) {
  constexpr int NM = GATE ? 2 : 1;
  constexpr int MP = 8 * MT;
  constexpr int U = GATE ? 2 : 4;      // chunks in flight per warp
  constexpr int GPC = kChunk / G;      // groups per chunk
  constexpr int WPG = 4 / GPC;         // words of a lane per group
  constexpr int RPO = kRows / CS;      // rows finished per CTA of the cluster
  constexpr int RP = MP + 2;           // pitch of the partial sums (even: float2 stores)
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const int xpitch = p.kslice + 32;    // elements: rows of x 64 bytes apart in the banks
  T* xs = reinterpret_cast<T*>(smem_raw);                                             // [MP][xpitch]
  float* red = reinterpret_cast<float*>(smem_raw + (size_t)MP * xpitch * sizeof(T));  // [NM][CS][RPO][RP]

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const uint32_t rank = cluster_rank();
  const int group = blockIdx.x / CS;
  const int row_lo = group * kRows + 16 * warp + r, row_hi = row_lo + 8;
  const bool v_lo = row_lo < p.N, v_hi = row_hi < p.N;
  const int k_begin = (int)rank * p.kslice;
  const int k_end = min(p.K, k_begin + p.kslice);
  const int nchunks = k_end > k_begin ? (k_end - k_begin + kChunk - 1) / kChunk : 0;

  cluster_arrive();
  // the CTA's weights on their way to L2 (nothing is read before the wait)
  for (int mtx = 0; mtx < NM; ++mtx) {
    const int lines = (max(k_end - k_begin, 0) / 2 + 127) / 128;
    for (int i = threadIdx.x; i < kRows * lines; i += kThreads) {
      const int row = group * kRows + i / lines;
      if (row < p.N) prefetch_l2(p.w[mtx] + (int64_t)row * p.ldw + k_begin / 2 + (i % lines) * 128);
    }
  }
  pdl_trigger();
  pdl_wait();

  const uint8_t* wp[NM][2];
  const T* sp[NM][2];
#pragma unroll
  for (int mtx = 0; mtx < NM; ++mtx) {
    wp[mtx][0] = p.w[mtx] + (int64_t)(v_lo ? row_lo : 0) * p.ldw + k_begin / 2 + 16 * c;
    wp[mtx][1] = p.w[mtx] + (int64_t)(v_hi ? row_hi : 0) * p.ldw + k_begin / 2 + 16 * c;
    const T* s = static_cast<const T*>(p.s[mtx]);
    sp[mtx][0] = s + (int64_t)(v_lo ? row_lo : 0) * p.lds + k_begin / G + c * GPC / 4;
    sp[mtx][1] = s + (int64_t)(v_hi ? row_hi : 0) * p.lds + k_begin / G + c * GPC / 4;
  }
  uint4 wv[U][NM][2];
  uint32_t sv[U][NM][2];  // scale of this lane's group of the chunk, as it is (converting it here would wait for it)
  auto load = [&](int u, int ch) {
    const bool in = ch < nchunks && k_begin + ch * kChunk + 32 * c < k_end;
#pragma unroll
    for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool ok = in && (h ? v_hi : v_lo);
        wv[u][mtx][h] = ok ? __ldcs(reinterpret_cast<const uint4*>(wp[mtx][h] + (int64_t)ch * (kChunk / 2)))
                           : make_uint4(0, 0, 0, 0);
        sv[u][mtx][h] = ok ? *reinterpret_cast<const unsigned short*>(sp[mtx][h] + (int64_t)ch * GPC) : 0;
      }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, u);

  // stage x[:, k_begin : k_end) (zero past M and k_end): 8 columns from
  // word_col(j, c) lie at 16-byte place 4 j + c of their chunk, in the order of the
  // pairs 0 4 1 5 2 6 3 7
  {
    const T* x = static_cast<const T*>(p.x);
    const int words = nchunks * (kChunk / 8);
    for (int i = threadIdx.x; i < MP * words; i += kThreads) {
      const int m = i / words, wd = i - m * words;
      const int place = wd % 16, ch = wd / 16;
      const int k = k_begin + ch * kChunk + word_col<G>(place / 4, place % 4);
      *reinterpret_cast<uint4*>(xs + (int64_t)m * xpitch + ch * kChunk + place * 8) =
          m < p.M && k < k_end ? pair_order(*reinterpret_cast<const uint4*>(x + (int64_t)m * p.ldx + k))
                               : make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();

  float acc[NM][MT][4];
#pragma unroll
  for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[mtx][t][e] = 0.f;

  const T* xl = xs + (int64_t)r * xpitch + 8 * c;
  for (int c0 = 0; c0 < nchunks; c0 += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = c0 + u;
      if (ch >= nchunks) break;
#pragma unroll
      for (int mtx = 0; mtx < NM; ++mtx) {
        uint32_t lo[4] = {wv[u][mtx][0].x, wv[u][mtx][0].y, wv[u][mtx][0].z, wv[u][mtx][0].w};
        uint32_t hi[4] = {wv[u][mtx][1].x, wv[u][mtx][1].y, wv[u][mtx][1].z, wv[u][mtx][1].w};
        spread<G>(lo, c);
        spread<G>(hi, c);
#pragma unroll
        for (int g = 0; g < GPC; ++g) {
          float part[MT][4];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[t][e] = 0.f;
#pragma unroll
          for (int jj = 0; jj < WPG; ++jj) {
            const int j = g * WPG + jj;
            uint32_t a[2][4];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              a[q][0] = Nib<T>::pair(lo[j], 2 * q);
              a[q][1] = Nib<T>::pair(hi[j], 2 * q);
              a[q][2] = Nib<T>::pair(lo[j], 2 * q + 1);
              a[q][3] = Nib<T>::pair(hi[j], 2 * q + 1);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const uint4 b = *reinterpret_cast<const uint4*>(xl + (int64_t)(8 * t) * xpitch + ch * kChunk + 32 * j);
              Nib<T>::mma(part[t], a[0], b.x, b.y);
              Nib<T>::mma(part[t], a[1], b.z, b.w);
            }
          }
          // lane quad + (4 / GPC) g holds the group's scales
          const int from = (lane & 28) + g * (4 / GPC);
          const float s_lo = scale_of<T>(GPC == 1 ? sv[u][mtx][0] : __shfl_sync(0xffffffffu, sv[u][mtx][0], from));
          const float s_hi = scale_of<T>(GPC == 1 ? sv[u][mtx][1] : __shfl_sync(0xffffffffu, sv[u][mtx][1], from));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            acc[mtx][t][0] = fmaf(part[t][0], s_lo, acc[mtx][t][0]);
            acc[mtx][t][1] = fmaf(part[t][1], s_lo, acc[mtx][t][1]);
            acc[mtx][t][2] = fmaf(part[t][2], s_hi, acc[mtx][t][2]);
            acc[mtx][t][3] = fmaf(part[t][3], s_hi, acc[mtx][t][3]);
          }
        }
      }
      load(u, ch + U);
    }
  }

  // partial sums to the CTA that finishes their rows
  cluster_wait();
  {
    const int owner = (16 * warp) / RPO;
    const int lrow = (16 * warp) % RPO + r;
#pragma unroll
    for (int mtx = 0; mtx < NM; ++mtx)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float* dst = red + ((int64_t)(mtx * CS + rank) * RPO + lrow + 8 * hf) * RP + 8 * t + 2 * c;
          st_cluster_f2(map_to_rank(dst, (uint32_t)owner), acc[mtx][t][2 * hf], acc[mtx][t][2 * hf + 1]);
        }
  }
  cluster_sync();
  T* y = static_cast<T*>(p.y);
  for (int i = threadIdx.x; i < RPO * p.M; i += kThreads) {
    const int m = i / RPO, lr = i % RPO;
    const int n = group * kRows + RPO * (int)rank + lr;
    if (n >= p.N) continue;
    float v[NM];
#pragma unroll
    for (int mtx = 0; mtx < NM; ++mtx) {
      v[mtx] = 0.f;
#pragma unroll
      for (int q = 0; q < CS; ++q) v[mtx] += red[((int64_t)(mtx * CS + q) * RPO + lr) * RP + m];
    }
    y[(int64_t)m * p.ldy + n] = from_f<T>(GATE ? silu_mul(v[0], v[NM - 1]) : v[0]);
  }
}

// The dense GEMM reads weights before griddepcontrol.wait, and these are fresh:
// no early trigger here, and a full dependency (a memset) between the two.
// 32 weights of a row per thread: 16-bit weights (q s, rounded once), row-major [N, K].
template <typename T>
__global__ void __launch_bounds__(256) w4_expand_kernel(const uint8_t* w, int64_t ldw, const T* s, int64_t lds, T* out,
                                                        int N, int K, int G) {
  pdl_wait();
  const int per = K / 32;
  const int64_t n = (int64_t)N * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per;
    const int k = (int)(i - row * per) * 32;
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(w + row * ldw + k / 2));
    const float sc = to_f<T>(s[row * lds + k / G]);
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
    T* dst = out + row * K + k;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      T o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = from_f<T>((float)((int)((words[j] >> (4 * e)) & 15u) - 8) * sc);
      *reinterpret_cast<uint4*>(dst + 8 * j) = *reinterpret_cast<const uint4*>(o);
    }
  }
}

size_t smem_bytes(int MT, bool gate, int kslice) {
  const int MP = 8 * MT;
  return (size_t)MP * (kslice + 32) * 2 + (size_t)(gate ? 2 : 1) * kRows * (MP + 2) * sizeof(float);
}
constexpr size_t kMaxSmem = 220 * 1024;
constexpr size_t kStreamSmem = 227 * 1024;

// CTAs that share K: from 17 rows on an eighth of it is too short to hide what
// comes before and after (12288 x 4096 gate and up, 32 rows: 70 us as 8, 46 as 4, 51
// as 2); below that few rows leave little else to do (4096 x 12288, 16 rows: 17 us
// as 8, 31 as 4).
constexpr int cluster_of(int MT) { return MT >= 4 ? 4 : 8; }
int kslice_of(int K, int cs) {
  const int per = (K + cs - 1) / cs;
  return (per + kChunk - 1) / kChunk * kChunk;
}

// Warps of the persistent kernel: as few as take the slices in as many rounds as 16 would.
int stream_warps(int K) {
  const int nsl = (K + kSlice - 1) / kSlice, rounds = (nsl + kStreamWarps - 1) / kStreamWarps;
  return (nsl + rounds - 1) / rounds;
}
bool stream_xreg(int K) { return (K + kSlice - 1) / kSlice <= kStreamWarps; }
size_t stream_smem(int M, int K, bool gate, int meet) {
  const int nm = gate ? 2 : 1, nw = stream_warps(K), nsl = (K + kSlice - 1) / kSlice;
  const bool xreg = stream_xreg(K);
  return (size_t)nw * stream_depth(gate, xreg) * nm * 2048 + (size_t)meet * sizeof(float) * nm * nw * 16 * ((M + 1) & ~1) +
         (xreg ? 0 : (size_t)M * (nsl * kSlice + 32) * 2 + (size_t)nsl * 8 * sizeof(float));
}
bool stream_fits(int M, int K, bool gate) {
  return M <= 16 && (M <= 8 || stream_xreg(K)) && stream_smem(M, K, gate, 1) <= kStreamSmem;
}

template <typename T, int MT, int G, bool GATE, bool XREG>
int launch_stream(const W4Params& p, cudaStream_t st) {
  auto kern = w4_stream_kernel<T, MT, G, GATE, XREG>;
  static bool configured[64] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return B200MM_ERR_DEVICE;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kStreamSmem) != cudaSuccess)
      return B200MM_ERR_LAUNCH;
    configured[dev] = true;
  }
  const int tiles = (p.N + 15) / 16, sms = num_sms(dev), grid = tiles < sms ? tiles : sms;
  // the warps meet as rarely as shared memory allows (one row, gate-up: 16.8 us with a meeting per
  // tile, 15.7 with one; 16 rows: fewer slots for three tiles a meeting took 29.8 instead of 28.1)
  int meet = MT == 1 ? (tiles + grid - 1) / grid : 1;
  while (meet > 1 && stream_smem(p.M, p.K, GATE, meet) > kStreamSmem) --meet;
  return launch_pdl(kern, dim3(grid), dim3(32 * stream_warps(p.K)), stream_smem(p.M, p.K, GATE, meet), st, p, meet) ==
                 cudaSuccess
             ? B200MM_OK
             : B200MM_ERR_LAUNCH;
}

template <typename T, int MT, int G, bool GATE, int CS>
int launch_w4(const W4Params& p, cudaStream_t st) {
  auto kern = w4_kernel<T, MT, G, GATE, CS>;
  const size_t smem = smem_bytes(MT, GATE, p.kslice);
  if (smem > kMaxSmem) return B200MM_ERR_SHAPE;
  static bool configured[64] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return B200MM_ERR_DEVICE;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem) != cudaSuccess)
      return B200MM_ERR_LAUNCH;
    configured[dev] = true;
  }
  const int groups = (p.N + kRows - 1) / kRows;
  return launch_pdl_cluster(kern, dim3(groups * CS), dim3(kThreads), smem, st, CS, p) == cudaSuccess ? B200MM_OK
                                                                                                  : B200MM_ERR_LAUNCH;
}

template <typename T, int MT, int G>
int launch_gate(const W4Params& p, bool gate, cudaStream_t st) {
  if constexpr (MT <= 2) {
    if (stream_fits(p.M, p.K, gate)) {
      if (stream_xreg(p.K))
        return gate ? launch_stream<T, MT, G, true, true>(p, st) : launch_stream<T, MT, G, false, true>(p, st);
      if constexpr (MT == 1)
        return gate ? launch_stream<T, 1, G, true, false>(p, st) : launch_stream<T, 1, G, false, false>(p, st);
    }
  }
  constexpr int CS = cluster_of(MT);
  return gate ? launch_w4<T, MT, G, true, CS>(p, st) : launch_w4<T, MT, G, false, CS>(p, st);
}
template <typename T, int MT>
int launch_group(const W4Params& p, int G, bool gate, cudaStream_t st) {
  if (G == 128) return launch_gate<T, MT, 128>(p, gate, st);
  if (G == 64) return launch_gate<T, MT, 64>(p, gate, st);
  return launch_gate<T, MT, 32>(p, gate, st);
}
template <typename T>
int launch_rows(const W4Params& p, int G, bool gate, cudaStream_t st) {
  if (p.M <= 8) return launch_group<T, 1>(p, G, gate, st);
  if (p.M <= 16) return launch_group<T, 2>(p, G, gate, st);
  if (p.M <= 32) return launch_group<T, 4>(p, G, gate, st);
  return launch_group<T, 8>(p, G, gate, st);
}

// Rows of x per launch: as many (a power of two from 8, at most 64) as leave room for the K slice in shared memory.
int rows_per_launch(const W4Args& a) {
  int m = kMaxRows;
  while (m > 8 && smem_bytes(m / 8, a.gate, kslice_of(a.K, cluster_of(m / 8))) > kMaxSmem) m /= 2;
  return m;
}

template <typename T>
int run_t(const W4Args& a) {
  if (a.M >= kDenseRows) {
    T* dense[3];
    for (int i = 0; i < 3; ++i) dense[i] = static_cast<T*>(a.ws) + i * (int64_t)a.N * a.K;
    for (int i = 0; i < (a.gate ? 2 : 1); ++i) {
      const int64_t want = ((int64_t)a.N * (a.K / 32) + 255) / 256;
      const unsigned grid = (unsigned)(want < 16384 ? want : 16384);
      if (launch_pdl(w4_expand_kernel<T>, dim3(grid), dim3(256), 0, a.stream, i ? a.w1 : a.w0, a.ldw,
                     static_cast<const T*>(i ? a.s1 : a.s0), a.lds, dense[i], a.N, a.K, a.G) != cudaSuccess)
        return B200MM_ERR_LAUNCH;
    }
    if (cudaMemsetAsync(dense[a.gate ? 2 : 1], 0, kFenceBytes, a.stream) != cudaSuccess) return B200MM_ERR_LAUNCH;
    DenseArgs d{};
    d.x = a.x; d.ldx = a.ldx; d.w0 = dense[0]; d.ldw0 = a.K;
    if (a.gate) { d.w1 = dense[1]; d.ldw1 = a.K; }
    d.y = a.y; d.ldy = a.ldy; d.M = a.M; d.N = a.N; d.K = a.K;
    d.dtype = a.dtype; d.gate = a.gate; d.stream = a.stream;
    return dense_dispatch(d);
  }
  const int step = rows_per_launch(a);
  for (int m0 = 0; m0 < a.M; m0 += step) {
    W4Params p{};
    p.x = static_cast<const T*>(a.x) + (int64_t)m0 * a.ldx; p.ldx = a.ldx;
    p.w[0] = a.w0; p.w[1] = a.w1; p.ldw = a.ldw;
    p.s[0] = a.s0; p.s[1] = a.s1; p.lds = a.lds;
    p.y = static_cast<T*>(a.y) + (int64_t)m0 * a.ldy; p.ldy = a.ldy;
    p.M = a.M - m0 < step ? a.M - m0 : step; p.N = a.N; p.K = a.K;
    p.kslice = kslice_of(a.K, cluster_of(p.M <= 8 ? 1 : p.M <= 16 ? 2 : 4));
    const int st = launch_rows<T>(p, a.G, a.gate, a.stream);
    if (st != B200MM_OK) return st;
  }
  return B200MM_OK;
}

}  // namespace

size_t w4_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gate) {
  return M >= kDenseRows ? (size_t)(gate ? 2 : 1) * N * K * 2 + kFenceBytes : 0;
}

int w4_run(const W4Args& a) {
  return a.dtype == B200MM_BF16 ? run_t<__nv_bfloat16>(a) : run_t<__half>(a);
}

}  // namespace b200mm
