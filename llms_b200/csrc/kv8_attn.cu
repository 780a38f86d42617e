// GQA decode attention (one query token per row) over the 8-bit KV cache:
//   out[b, h] = sum_t softmax_t(q[b, h] . kq[t] sk[t / 64] scale) vq[t] sv[t / 64],  t <= pos[b].
//
// The step streams 2 D bytes per cached token and KV head, half of what the
// 16-bit cache costs, so the arithmetic per byte doubles; the kernel keeps the
// stream in flight and the instructions per byte few:
//   * a warp is on its own.  The flattened sequence of units (64 tokens, or 16
//     where there are few) over (row, KV head, context) is cut into one
//     contiguous range per warp, eight warps to a CTA and one CTA per SM.  The
//     lengths are read on the device, so one captured graph serves every
//     position, and rows of any length share the machine evenly;
//   * each warp fills a private ring of three slots with cp.async (K of a
//     block, V of a block, alternately): two slots in flight while one is
//     computed, 128 KB per SM, with no barrier between warps.  16-byte chunks
//     are swizzled so that the fragment loads below meet no bank twice;
//   * tokens are the rows of the matrix instructions (m16n8k16, fp16 x fp16 ->
//     fp32) and the group's query heads the 8 columns: S[t, h] = K[t, d] Q[d, h]
//     and O[d, h] = V^T[d, t] P[t, h].  8-bit values become fp16 exactly in
//     registers.  The order of d inside a product is free, so a lane takes 16
//     bytes of a token row as they lie; pairs of tokens for V^T are picked
//     from two rows by the byte permute that widens them;
//   * q is scaled per head by a power of two that brings its largest element
//     into [2^14, 2^15): bf16 -> fp16 is then exact to 2^-38 of that element;
//   * the softmax is local to a block: p = 2^(s - max of the block + 14),
//     rounded to fp16 (11 bits, and 2^-38 of the block's largest still counts),
//     the block's O in fp32, joined to the running sums with one factor
//     that also carries the block's scale of V.
// Each warp has one partial (max, sum, O) per (row, head) that its range touches.
// Those of a CTA's warps that end in the same pair are joined in shared memory
// (one long row of 8 KV heads: 18 partials per pair instead of 148, and 15 -> 4
// us for the second kernel, which joins the rest).
//
// Other shapes (fp32, head dims other than 64 / 128, more than 16 query heads
// per KV head) run a kernel of one CTA per (head, row) on plain arithmetic.
#include "kv8.cuh"

namespace b200mm {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlots = 3;       // ring slots per warp
constexpr int kMaxRows = 1024;  // rows of one launch (their lengths are summed by one CTA)
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  b200mm_kv8 c;
  const void* q; int64_t q_sb, q_sh;
  void* out; int64_t o_sb, o_sh;
  int B, H, g;  // g = H / KV
  Kv8Pos pos;
  float scale;
  int W;        // warps of the split kernel
  float* pacc;  // [W + B KV][g][D]: O, relative to the partial's max
  float* pml;   // [W + B KV][g][2]: max (log2 units), sum
};

// The work of a launch: T units of `ut` tokens, flattened over (row, KV head,
// context); warp i of W (no more than there are units, so that no range is
// empty) takes [i T / W, (i + 1) T / W).  Partials of warp i for pair
// p = row KV + head go to slot i + p, distinct for every (i, p) that meet
// (ranges are contiguous); a warp that ends in the pair in which the one before
// it in its CTA ends has its partial joined to that one's.  Units are whole blocks once every warp has two of
// them, and 16 tokens below that, so that short contexts spread over the SMs.
struct Plan {
  int64_t T;
  int ut, W;
};
__device__ __forceinline__ int units(int len, int ut) { return (len + ut - 1) / ut; }
__device__ __forceinline__ Plan make_plan(int64_t n64, int64_t n16, int W) {
  if (n64 >= 2 * (int64_t)W) return Plan{n64, 64, W};
  return Plan{n16, 16, n16 < W ? (int)n16 : W};
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_h(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Byte offset of 16-byte chunk `c` of token row `row` in a slot.  Rows of 128
// bytes: K fragments read rows 2i, 2i + 1 together (chunks c..c + 3 of each),
// V fragments rows 0, 2, 4, 6 (+ const) together (two neighbouring chunks of
// each).  Rows of 64 bytes lie two to a 128-byte line.
template <int D, bool V>
__device__ __forceinline__ uint32_t slot_off(int row, int c) {
  if constexpr (D == 128) {
    const int x = V ? ((row >> 1) & 3) << 1 : (row & 1) << 2;
    return (uint32_t)(row * 128 + ((c ^ x) << 4));
  } else {
    const int x = ((row >> 1) & 3) << 1;
    return (uint32_t)((row >> 1) * 128 + (((((row & 1) << 2) | c) ^ x) << 4));
  }
}

// A part of one block, at most 64 tokens of one pair.
struct Seg {
  int b, kvh, blk;
  int s0, s1;   // 16-token steps [s0, s1) of the block
  int valid;    // tokens of the block inside the context
  float sk, sv;
};

template <typename T, int D, int NH>
__global__ void __launch_bounds__(kThreads, 1) kv8_split_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int J = D / 64;             // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;            // m-tiles of O^T
  constexpr uint32_t SLOT = 64 * D;     // bytes
  constexpr int CPR = D / 16;           // 16-byte chunks per row
  constexpr int RPI = 32 / CPR;         // rows per warp-wide copy
  extern __shared__ __align__(1024) unsigned char ring[];
  __shared__ int pre[kMaxRows + 1];     // units of one head in rows before b
  __shared__ long long red[2][kWarps];
  __shared__ int last_s[kWarps];        // the pair that a warp's range ends in

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  pdl_trigger();
  pdl_wait();

  // the plan: lengths summed over the rows
  const int KV = a.c.KV;
  Plan plan;
  {
    constexpr int PT = kMaxRows / kThreads;
    int len[PT];
    long long n64 = 0, n16 = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int b = threadIdx.x * PT + i;
      len[i] = b < a.B ? kv8_len(a.pos(b), a.c.S) : 0;
      n64 += units(len[i], 64);
      n16 += units(len[i], 16);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      n64 += __shfl_xor_sync(0xffffffffu, n64, o);
      n16 += __shfl_xor_sync(0xffffffffu, n16, o);
    }
    if (lane == 0) {
      red[0][warp] = n64;
      red[1][warp] = n16;
    }
    __syncthreads();
    n64 = n16 = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      n64 += red[0][w];
      n16 += red[1][w];
    }
    plan = make_plan(n64 * KV, n16 * KV, a.W);
    __syncthreads();
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) mine += units(len[i], plan.ut);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) red[0][warp] = inc;
    __syncthreads();
    int base = inc - mine;
    for (int w = 0; w < warp; ++w) base += (int)red[0][w];
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      pre[threadIdx.x * PT + i] = base;
      base += units(len[i], plan.ut);
    }
    if (threadIdx.x == kThreads - 1) pre[kMaxRows] = base;
    __syncthreads();
  }
  const int wi = blockIdx.x * kWarps + warp;
  int last_pair = -1;  // none: the warp has no work
  // state of the running pair
  uint32_t qf[NH][J][4][2];  // B fragments of q
  float qinv[NH][2];         // 1 / q's power of two, heads 2c, 2c + 1 (times scale, log2 units)
  float o[NH][MT][4];
  float m[NH][2], l[NH][2];  // max and this lane's sum, heads 2c, 2c + 1
  auto end_pair = [&](float* acc, float* ml) {  // the partial of the pair: [g][D], [g][2]
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float sum = l[n][k];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int h = 8 * n + 2 * c + k;
        if (h < a.g) {
          // m-tile i holds d = 2 MT r' + 2i (rows r' = r) and + 1 (rows r + 8)
          float* dst = acc + h * D + 2 * MT * r;
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) =
                make_float4(o[n][i][k], o[n][i][2 + k], o[n][i + 1][k], o[n][i + 1][2 + k]);
          if (r == 0) *reinterpret_cast<float2*>(ml + h * 2) = make_float2(m[n][k], sum);
        }
      }
  };

  if (wi < plan.W) {
  const int64_t u0 = (int64_t)wi * plan.T / plan.W, u1 = (int64_t)(wi + 1) * plan.T / plan.W;

  // ---- the load cursor: next segment at unit `un` of pair (nb, nh) ----
  int nb, nh, un, nu;
  int64_t rem = u1 - u0;
  {
    int lo = 0, hi = a.B - 1;  // the last row with KV pre[row] <= u0 (it is not empty)
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if ((int64_t)pre[m] * KV <= u0) lo = m; else hi = m - 1;
    }
    nb = lo;
    nu = pre[nb + 1] - pre[nb];
    const int64_t v = u0 - (int64_t)pre[nb] * KV;
    nh = (int)(v / nu);
    un = (int)(v - (int64_t)nh * nu);
  }
  auto next_seg = [&](Seg& s) -> bool {
    if (rem <= 0) return false;
    if (un == nu) {  // next pair; rows without tokens have none
      un = 0;
      if (++nh == KV) {
        nh = 0;
        do { ++nb; } while (pre[nb + 1] == pre[nb]);
        nu = pre[nb + 1] - pre[nb];
      }
    }
    const int len = kv8_len(a.pos(nb), a.c.S);
    const int t = un * plan.ut;
    s.b = nb;
    s.kvh = nh;
    s.blk = t >> 6;
    s.valid = min(64, len - (s.blk << 6));
    int n = plan.ut == 64 ? 1 : 4 - ((t & 63) >> 4);  // units left in this block
    n = min(n, nu - un);
    if (n > rem) n = (int)rem;
    s.s0 = (t & 63) >> 4;
    s.s1 = min(s.s0 + (n * plan.ut >> 4), (s.valid + 15) >> 4);
    un += n;
    rem -= n;
    const int64_t o = (int64_t)s.b * a.c.s_sb + (int64_t)s.kvh * a.c.s_sh + s.blk;
    s.sk = a.c.ks[o];
    s.sv = a.c.vs[o];
    return true;
  };

  unsigned char* my = ring + (size_t)warp * kSlots * SLOT;
  const uint32_t my_u = static_cast<uint32_t>(__cvta_generic_to_shared(my));
  auto issue = [&](const Seg& s, bool is_v, int slot) {
    const int8_t* src = (is_v ? a.c.vq : a.c.kq) + (int64_t)s.b * a.c.q_sb + (int64_t)s.kvh * a.c.q_sh +
                        (int64_t)s.blk * (64 * D) + lane * 16;
    const uint32_t dst = my_u + slot * SLOT;
#pragma unroll
    for (int i = 0; i < 64 / RPI; ++i) {
      const int row = i * RPI + lane / CPR, ch = lane % CPR;
      const int st = i * RPI / 16;
      if (st >= s.s0 && st < s.s1)
        cp_async16(dst + (is_v ? slot_off<D, true>(row, ch) : slot_off<D, false>(row, ch)), src + i * 512);
    }
  };

  auto begin_pair = [&](const Seg& s) {
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int h = 8 * n + r;
      const T* qp = static_cast<const T*>(a.q) + (int64_t)s.b * a.q_sb + ((int64_t)s.kvh * a.g + h) * a.q_sh + 16 * c;
      float f[J][16];
      float mx = 0.f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (h < a.g) v = *reinterpret_cast<const uint4*>(qp + 64 * j + 8 * e);
          Chunk<T>::unpack(v, &f[j][8 * e]);
        }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          mx = fmaxf(mx, fabsf(f[j][e]));
          bad |= !(fabsf(f[j][e]) < INFINITY);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 28)) & 15;
      // 2^(14 - exponent of the largest), kept where it and its inverse are normal
      const int e = min(268 - (int)(__float_as_uint(mx) >> 23), 253);
      const float up = __uint_as_float((uint32_t)max(e, 1) << 23), down = __uint_as_float((uint32_t)(254 - max(e, 1)) << 23);
      float inv = bad ? __int_as_float(0x7fc00000) : down;  // an infinity or NaN in q: the head is NaN
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          qf[n][j][w][0] = pack_h2(f[j][4 * w] * up, f[j][4 * w + 1] * up);
          qf[n][j][w][1] = pack_h2(f[j][4 * w + 2] * up, f[j][4 * w + 3] * up);
        }
      qinv[n][0] = __shfl_sync(0xffffffffu, inv, 8 * c) * (a.scale * kLog2e);
      qinv[n][1] = __shfl_sync(0xffffffffu, inv, 8 * c + 4) * (a.scale * kLog2e);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
  };
  Seg cur, nxt;
  bool more = next_seg(cur);  // a range is not empty
  int slot = 0;               // of cur's K; its V is in the next one
  issue(cur, false, 0);
  cp_commit();
  issue(cur, true, 1);
  cp_commit();
  begin_pair(cur);
  while (true) {
    more = next_seg(nxt);
    const int slot_v = slot + 1 == kSlots ? 0 : slot + 1;
    const int slot_n = slot_v + 1 == kSlots ? 0 : slot_v + 1;
    if (more) issue(nxt, false, slot_n);
    cp_commit();
    cp_wait<2>();  // cur's K
    __syncwarp();

    // ---- S = K Q ----
    float sc[NH][4][4];
    {
      const uint32_t kb = my_u + slot * SLOT;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][s][e] = 0.f;
        if (s >= cur.s0 && s < cur.s1) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint4 lo = lds16(kb + slot_off<D, false>(16 * s + r, 4 * j + c));
            const uint4 hi = lds16(kb + slot_off<D, false>(16 * s + r + 8, 4 * j + c));
            const uint32_t L[4] = {lo.x ^ 0x80808080u, lo.y ^ 0x80808080u, lo.z ^ 0x80808080u, lo.w ^ 0x80808080u};
            const uint32_t G[4] = {hi.x ^ 0x80808080u, hi.y ^ 0x80808080u, hi.z ^ 0x80808080u, hi.w ^ 0x80808080u};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t a0 = i8x2_to_h2(L[w], 0), a1 = i8x2_to_h2(G[w], 0);
              const uint32_t a2 = i8x2_to_h2(L[w], 1), a3 = i8x2_to_h2(G[w], 1);
#pragma unroll
              for (int n = 0; n < NH; ++n) mma_h(sc[n][s], a0, a1, a2, a3, qf[n][j][w][0], qf[n][j][w][1]);
            }
          }
        }
      }
    }
    __syncwarp();
    // cur's K slot is free: nxt's V
    if (more) issue(nxt, true, slot);
    cp_commit();

    // ---- the block's softmax; tokens outside [16 s0, valid) do not count ----
    uint32_t pf[NH][4][2];
    float fo[NH][2], fb[NH][2];  // factors of the running and of the block's sums
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float mb[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 16 * s + r + 8 * (e >> 1);
          const bool on = s >= cur.s0 && s < cur.s1 && t < cur.valid;
          const float v = on ? sc[n][s][e] * (qinv[n][e & 1] * cur.sk) : -INFINITY;
          sc[n][s][e] = v;
          mb[e & 1] = fmaxf(mb[e & 1], v);
        }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 4));
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 8));
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 16));
        if (mb[k] == -INFINITY) mb[k] = 0.f;  // no finite score: p is 0 (or NaN where a score is)
        const float mn = fmaxf(m[n][k], mb[k]);
        fo[n][k] = ex2(m[n][k] - mn);
        fb[n][k] = ex2(mb[k] - mn);
        m[n][k] = mn;
      }
      float lb[2] = {0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = ex2(sc[n][s][e] - (mb[e & 1] - 14.f));
          lb[e & 1] += p[e];
        }
        pf[n][s][0] = transpose8x8(pack_h2(p[0], p[1]));  // tokens 2c, 2c + 1 of head r
        pf[n][s][1] = transpose8x8(pack_h2(p[2], p[3]));  // tokens 2c + 8, 2c + 9
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        l[n][k] = l[n][k] * fo[n][k] + lb[k] * fb[n][k];
        fb[n][k] *= cur.sv;
      }
    }

    cp_wait<2>();  // cur's V
    __syncwarp();
    // ---- O = O fo + (V^T P) fb ----
    {
      const uint32_t vb = my_u + slot_v * SLOT;
      float ob[NH][MT][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) ob[n][i][e] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s >= cur.s0 && s < cur.s1) {
          const int t = 16 * s + 2 * c;
          uint32_t v0[MT / 2], v1[MT / 2], v8[MT / 2], v9[MT / 2];  // 2 MT bytes of four tokens, from d = 2 MT r
          auto load = [&](uint32_t* dst, int row) {
            if constexpr (D == 128) {
              const uint4 x = lds16(vb + slot_off<D, true>(row, r));
              dst[0] = x.x; dst[1] = x.y; dst[2] = x.z; dst[3] = x.w;
            } else {
              const uint2 x = lds8(vb + slot_off<D, true>(row, r >> 1) + 8 * (r & 1));
              dst[0] = x.x; dst[1] = x.y;
            }
          };
          load(v0, t);
          load(v1, t + 1);
          load(v8, t + 8);
          load(v9, t + 9);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int w = i >> 1, k = 2 * (i & 1);
            const uint32_t a0 = i8_pair_to_h2(v0[w], v1[w], k), a1 = i8_pair_to_h2(v0[w], v1[w], k + 1);
            const uint32_t a2 = i8_pair_to_h2(v8[w], v9[w], k), a3 = i8_pair_to_h2(v8[w], v9[w], k + 1);
#pragma unroll
            for (int n = 0; n < NH; ++n) mma_h(ob[n][i], a0, a1, a2, a3, pf[n][s][0], pf[n][s][1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][i][e] = o[n][i][e] * fo[n][e & 1] + ob[n][i][e] * fb[n][e & 1];
    }
    __syncwarp();
    if (!more) break;
    if (nxt.b != cur.b || nxt.kvh != cur.kvh) {
      const int64_t at = ((int64_t)wi + (int64_t)cur.b * KV + cur.kvh) * a.g;
      end_pair(a.pacc + at * D, a.pml + at * 2);
      begin_pair(nxt);
    }
    cur = nxt;
    slot = slot_n;
  }
  cp_wait<0>();
  last_pair = cur.b * KV + cur.kvh;
  }  // (warps with work)

  // ---- the last partials of the CTA's warps, joined where they are of one pair ----
  __syncthreads();  // the rings are empty
  float* sacc = reinterpret_cast<float*>(ring);          // [warp][g][D]
  float* sml = sacc + (size_t)kWarps * a.g * D;          // [warp][g][2]
  if (last_pair >= 0) end_pair(sacc + (size_t)warp * a.g * D, sml + warp * a.g * 2);
  if (lane == 0) last_s[warp] = last_pair;
  __syncthreads();
  for (int i = threadIdx.x; i < kWarps * a.g * (D / 4); i += kThreads) {
    const int d = i % (D / 4) * 4, h = i / (D / 4) % a.g, w0 = i / (D / 4) / a.g;
    const int pair = last_s[w0];
    if (pair < 0 || (w0 > 0 && last_s[w0 - 1] == pair)) continue;  // no work, or joined to the one before
    int w1 = w0 + 1;
    float mx = sml[(w0 * a.g + h) * 2];
    for (; w1 < kWarps && last_s[w1] == pair; ++w1) mx = fmaxf(mx, sml[(w1 * a.g + h) * 2]);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int q = w0; q < w1; ++q) {
      const float2 ml = *reinterpret_cast<const float2*>(sml + (q * a.g + h) * 2);
      const float f = ml.x == mx ? 1.f : ex2(ml.x - mx);
      const float4 o4 = *reinterpret_cast<const float4*>(sacc + ((size_t)q * a.g + h) * D + d);
      v.x = fmaf(o4.x, f, v.x); v.y = fmaf(o4.y, f, v.y); v.z = fmaf(o4.z, f, v.z); v.w = fmaf(o4.w, f, v.w);
      l = fmaf(ml.y, f, l);
    }
    const int64_t at = ((int64_t)blockIdx.x * kWarps + w0 + pair) * a.g + h;
    *reinterpret_cast<float4*>(a.pacc + at * D + d) = v;
    if (d == 0) *reinterpret_cast<float2*>(a.pml + at * 2) = make_float2(mx, l);
  }
}

// ---------------------------------------------------------------------------
// join: out[b, h] = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k over the
// partials of the pair.  grid (H, B), 8 warps over the partials, lane = 4 dims.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) kv8_join_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float acc_s[kWarps][128];
  __shared__ float m_s[kWarps], l_s[kWarps];
  __shared__ long long red[4][kWarps];
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / a.g, hl = h % a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.c.D, KV = a.c.KV;
  pdl_trigger();
  pdl_wait();
  long long s[4] = {0, 0, 0, 0};  // units of 64 and of 16 tokens, over all rows and over the rows before b
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const int len = kv8_len(a.pos(i), a.c.S);
    s[0] += units(len, 64);
    s[1] += units(len, 16);
    if (i < b) {
      s[2] += units(len, 64);
      s[3] += units(len, 16);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
    if (lane == 0) red[k][warp] = s[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    s[k] = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s[k] += red[k][w];
  }
  const int len = kv8_len(a.pos(b), a.c.S);
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  if (len == 0) {  // a row that is not there
    for (int d = threadIdx.x; d < D; d += kThreads) out[d] = from_f<T>(0.f);
    return;
  }
  const Plan plan = make_plan(s[0] * KV, s[1] * KV, a.W);
  const int64_t nu = units(len, plan.ut);
  const int64_t lo = (plan.ut == 64 ? s[2] : s[3]) * KV + kvh * nu, hi = lo + nu;
  const int i0 = (int)(((lo + 1) * plan.W - 1) / plan.T), i1 = (int)((hi * plan.W - 1) / plan.T);  // lo, hi - 1
  const int64_t p = (int64_t)b * KV + kvh;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool mine = 4 * lane < D;
  // partials: warp i0's, the first of each later CTA, and warp i1's if it goes on to the next pair
  // (otherwise it ends here, as all between do, and is joined to its CTA's)
  const int first = (i0 / kWarps + 1) * kWarps;
  const int later = i1 < first ? 0 : (i1 - first) / kWarps + 1;
  const bool own = i1 > i0 && i1 % kWarps != 0 && (int64_t)(i1 + 1) * plan.T / plan.W > hi;
#pragma unroll 4
  for (int k = warp; k < 1 + later + (own ? 1 : 0); k += kWarps) {
    const int i = k == 0 ? i0 : k <= later ? first + (k - 1) * kWarps : i1;
    const int64_t slot = (i + p) * a.g + hl;
    const float2 ml = *reinterpret_cast<const float2*>(a.pml + slot * 2);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) v = *reinterpret_cast<const float4*>(a.pacc + slot * D + 4 * lane);
    const float mn = fmaxf(m, ml.x), f0 = m == mn ? 1.f : ex2(m - mn), f1 = ml.x == mn ? 1.f : ex2(ml.x - mn);
    acc.x = acc.x * f0 + v.x * f1;
    acc.y = acc.y * f0 + v.y * f1;
    acc.z = acc.z * f0 + v.z * f1;
    acc.w = acc.w * f0 + v.w * f1;
    l = l * f0 + ml.y * f1;
    m = mn;
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  if (mine) *reinterpret_cast<float4*>(&acc_s[warp][4 * lane]) = acc;
  __syncthreads();
  if (threadIdx.x < D) {
    float mm = m_s[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, m_s[w]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m_s[w] == -INFINITY ? 0.f : ex2(m_s[w] - mm);
      num += acc_s[w][threadIdx.x] * f;
      den += l_s[w] * f;
    }
    out[threadIdx.x] = from_f<T>(num / den);
  }
}

// ---------------------------------------------------------------------------
// any shape: one CTA per (head, row), a warp per token, D <= 256
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) kv8_generic_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int E = 8;  // dims per lane
  __shared__ float acc_s[kWarps][256];
  __shared__ float m_s[kWarps], l_s[kWarps];
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / a.g, D = a.c.D;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  const int len = kv8_len(a.pos(b), a.c.S);
  const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;
  const int64_t base = (int64_t)b * a.c.q_sb + (int64_t)kvh * a.c.q_sh;
  const int64_t sbase = (int64_t)b * a.c.s_sb + (int64_t)kvh * a.c.s_sh;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  float qv[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < D ? to_f<T>(q[d]) : 0.f;
    acc[e] = 0.f;
  }
  for (int64_t t = warp; t < len; t += kWarps) {
    const int8_t* kr = a.c.kq + base + t * D;
    const int8_t* vr = a.c.vq + base + t * D;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < D) s = fmaf(qv[e], (float)kr[lane + 32 * e], s);
    s = warp_sum(s) * (a.c.ks[sbase + t / kKv8Block] * (a.scale * kLog2e));
    const float mn = fmaxf(m, s), f = m == mn ? 1.f : exp2f(m - mn), p = exp2f(s - (mn == -INFINITY ? 0.f : mn));
    const float pv = p * a.c.vs[sbase + t / kKv8Block];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < D) acc[e] = acc[e] * f + pv * (float)vr[lane + 32 * e];
    l = l * f + p;
    m = mn;
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < D) acc_s[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  if (threadIdx.x < D) {
    float mm = m_s[0];
    for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, m_s[w]);
    float num = 0.f, den = 0.f;
    for (int w = 0; w < kWarps; ++w) {
      const float f = m_s[w] == -INFINITY ? 0.f : exp2f(m_s[w] - mm);
      num += acc_s[w][threadIdx.x] * f;
      den += l_s[w] * f;
    }
    out[threadIdx.x] = from_f<T>(len == 0 ? 0.f : num / den);
  }
}

bool fast_shape(const b200mm_kv8& c, int H) {
  return c.dtype != B200MM_F32 && (c.D == 64 || c.D == 128) && H / c.KV <= 16;
}

// CTAs of the split kernel: one per SM, fewer where the capacity has no work for them
int split_ctas(const b200mm_kv8& c, int rows) {
  const int64_t most = (int64_t)rows * c.KV * ((c.S + 15) / 16);
  const int64_t need = (most + kWarps - 1) / kWarps;
  const int sms = num_sms(current_device());
  return (int)(need < sms ? need : sms);
}

template <typename T, int D, int NH>
int launch_split(const AttnArgs& a) {
  constexpr size_t smem = (size_t)kWarps * kSlots * 64 * D;
  auto kern = kv8_split_kernel<T, D, NH>;
  const int dev = current_device();
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64) return B200MM_ERR_DEVICE;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return B200MM_ERR_LAUNCH;
    configured[dev] = true;
  }
  return B200MM_OK;
}

template <typename T, int D, int NH>
int run_fast(const AttnArgs& a, cudaStream_t st) {
  const int s = launch_split<T, D, NH>(a);
  if (s != B200MM_OK) return s;
  constexpr size_t smem = (size_t)kWarps * kSlots * 64 * D;
  cudaError_t e = launch_pdl(kv8_split_kernel<T, D, NH>, dim3(a.W / kWarps), dim3(kThreads), smem, st, a);
  if (e != cudaSuccess) return B200MM_ERR_LAUNCH;
  e = launch_pdl(kv8_join_kernel<T>, dim3(a.H, a.B), dim3(kThreads), 0, st, a);
  return e == cudaSuccess ? B200MM_OK : B200MM_ERR_LAUNCH;
}

template <typename T>
int run(const AttnArgs& a, bool fast, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (fast) {
      if (a.c.D == 128) return a.g <= 8 ? run_fast<T, 128, 1>(a, st) : run_fast<T, 128, 2>(a, st);
      return a.g <= 8 ? run_fast<T, 64, 1>(a, st) : run_fast<T, 64, 2>(a, st);
    }
  }
  return launch_pdl(kv8_generic_kernel<T>, dim3(a.H, a.B), dim3(kThreads), 0, st, a) == cudaSuccess
             ? B200MM_OK
             : B200MM_ERR_LAUNCH;
}

}  // namespace

size_t kv8_decode_workspace_bytes(const b200mm_kv8& c, int B, int H) {
  if (!fast_shape(c, H)) return 0;
  const int rows = B < kMaxRows ? B : kMaxRows;
  const size_t slots = (size_t)split_ctas(c, rows) * kWarps + (size_t)rows * c.KV;
  return slots * (H / c.KV) * (c.D + 2) * sizeof(float);
}

int kv8_decode(const b200mm_kv8& c, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
               int B, int H, Kv8Pos pos, float scale, void* ws, cudaStream_t st) {
  const bool fast = fast_shape(c, H) && !g_force_generic.load(std::memory_order_relaxed);
  const int esz = c.dtype == B200MM_F32 ? 4 : 2;
  for (int b0 = 0; b0 < B; b0 += kMaxRows) {
    AttnArgs a{};
    a.c = c;
    a.c.kq += (int64_t)b0 * c.q_sb;
    a.c.vq += (int64_t)b0 * c.q_sb;
    a.c.ks += (int64_t)b0 * c.s_sb;
    a.c.vs += (int64_t)b0 * c.s_sb;
    a.q = static_cast<const char*>(q) + (int64_t)b0 * q_sb * esz;
    a.out = static_cast<char*>(out) + (int64_t)b0 * o_sb * esz;
    a.q_sb = q_sb; a.q_sh = q_sh; a.o_sb = o_sb; a.o_sh = o_sh;
    a.B = B - b0 < kMaxRows ? B - b0 : kMaxRows;
    a.H = H;
    a.g = H / c.KV;
    a.pos = pos;
    if (pos.dev) a.pos.dev += (int64_t)b0 * pos.stride;
    a.scale = scale;
    if (fast) {
      a.W = split_ctas(c, a.B) * kWarps;
      const int64_t slots = (int64_t)a.W + (int64_t)a.B * c.KV;
      a.pacc = static_cast<float*>(ws);
      a.pml = a.pacc + slots * a.g * c.D;
    }
    int s;
    if (c.dtype == B200MM_BF16) s = run<__nv_bfloat16>(a, fast, st);
    else if (c.dtype == B200MM_F16) s = run<__half>(a, fast, st);
    else s = run<float>(a, fast, st);
    if (s != B200MM_OK) return s;
  }
  return B200MM_OK;
}

}  // namespace b200mm
