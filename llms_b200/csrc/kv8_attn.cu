// GQA decode attention (one query token per row) over the 8-bit KV cache:
//   out[b, h] = sum_t softmax_t(q[b, h] . kq[t] sk[t / 64] scale) vq[t] sv[t / 64],  t <= pos[b].
//
// The step streams 2 D bytes per cached token and KV head, half of what the
// 16-bit cache costs, so the arithmetic per byte doubles; the kernel keeps the
// stream in flight and the instructions per byte few:
//   * a warp is on its own.  The flattened sequence of units (64 tokens, or 16
//     where there are too few of them) over (row, KV head, context) is cut into one
//     contiguous range per warp, twelve warps to a CTA and one CTA per SM.  The
//     lengths are read on the device, so one captured graph serves every
//     position, and rows of any length share the machine evenly;
//   * each warp has two slots of its own, for K and for V of a block, and fills
//     each with cp.async for the next block as soon as it has used it: the other
//     is in flight meanwhile, 96 to 192 KB per SM, with no barrier between warps.
//     16-byte chunks are swizzled so that the fragment loads below meet no bank twice;
//   * tokens are the rows of the matrix instructions (m16n8k16, fp16 x fp16 ->
//     fp32) and the group's query heads the 8 columns: S[t, h] = K[t, d] Q[d, h]
//     and O[d, h] = V^T[d, t] P[t, h].  8-bit values become fp16 exactly in
//     registers.  The order of d inside a product is free, so a lane takes 16
//     bytes of a token row as they lie; pairs of tokens for V^T are picked
//     from two rows by the byte permute that widens them;
//   * q is scaled per head by a power of two that brings its largest element
//     into [2^14, 2^15): bf16 -> fp16 is then exact to 2^-38 of that element;
//   * the softmax is local to a block: p = 2^(s - max of the block + 14), held
//     as two fp16 numbers, p rounded and what that left (22 bits; 2^-39 of the
//     block's largest still counts).  Both multiply V into the block's O in fp32,
//     which is joined to the running sums with one factor that also carries the
//     block's scale of V.  (p in one fp16 number would cost fp16 outputs nearly as
//     much as their own rounding does: 2.6e-4 off the formula, by the norm, where the
//     rounding alone is 2.1e-4.)
// Each warp has one partial (max, sum, O) per (row, head) that its range touches.
// Those of a CTA's warps that end in the same pair are joined in shared memory
// (one long row of 8 KV heads: the 222 warps of a pair leave 19 or 20), and a
// second kernel joins the rest.
//
// Measured (B200, bf16, H 32, KV 8, D 128; attention, and the step with its append):
// 16 rows of 32768 tokens 165 us, 6.5 TB/s of cache, 171-178 the step; 32 rows of 4096
// 52.6 us (5.1 TB/s) and 58, of 1..4096 at random 37.7 (3.9) and 42; 1 row of 32768
// 23.4 (2.9) and 26.8, of 512 8.9 and 11.5 (the append runs beside the attention, but
// its CTAs and the attention's do not fit on one SM).  Long contexts are bound by HBM (at
// 16 x 32768 the schedulers issue in 66 % of the cycles, so not by much); short ones by
// what does not shrink: two dependent launches, the plan, one block's latency and the
// joins, 8 us; those between by whole blocks per warp (1 x 32768: 4096 blocks for 1776
// warps, three rounds).
//
// Other shapes (fp32, head dims other than 64 / 128, more than 16 query heads
// per KV head) run a kernel of one CTA per (head, row) on plain arithmetic.
#include "kv8.cuh"

namespace b200mm {

namespace {

constexpr int kGenericThreads = 256;
constexpr int kGenericWarps = kGenericThreads / 32;
constexpr int kMaxRows = 1024;  // rows of one launch (their lengths are summed by one CTA)
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  b200mm_kv8 c;
  const void* q; int64_t q_sb, q_sh;
  void* out; int64_t o_sb, o_sh;
  int B, H, g;  // g = H / KV
  Kv8Pos pos;
  float scale;
  bool early;   // right behind the append of one token: only the rows' last blocks wait for it
  int W, cw;    // warps of the split kernel, and of a CTA of it
  float* pacc;  // [W + B KV][g][D]: sum of p v, relative to the partial's max
  float* pml;   // [W + B KV][g][2]: max (log2 units), sum
};

// The work of a launch: T units of 2^lg tokens, flattened over (row, KV head,
// context); warp i of W (no more than there are units, so that no range is
// empty) takes T / W of them, the first T mod W warps one more.  Partials of
// warp i for pair p = row KV + head go to slot i + p, distinct for every (i, p)
// that meet (ranges are contiguous); a warp that ends in the pair in which the
// one before it in its CTA ends has its partial joined to that one's.  Units are
// whole blocks: a part of a block costs a warp nearly what the block does, so
// finer ranges are even and no shorter (a step of 1 x 32768 with units of 16
// tokens 27.3 us instead of 25.8, of 1 x 4096 15.5 instead of 12.2, of 32 x 2048
// ragged 38.0 instead of 28.6).  Below a block for every fourth warp they are 16
// tokens, so that short contexts spread over the SMs (1 x 512: 11.1 us, 12.2 with
// blocks; 16 x 128: 14.5, 16.4).
// (T fits 32 bits: 2^31 blocks would be 2 TB of cache.)
struct Plan {
  int T, lg, W, per, more;  // per = T / W, more = T mod W
  __device__ __forceinline__ int begin(int i) const { return i * per + min(i, more); }
  __device__ __forceinline__ int warp_of(int u) const {
    const int cut = more * (per + 1);
    return u < cut ? u / (per + 1) : more + (u - cut) / per;
  }
};
__device__ __forceinline__ int units(int len, int lg) { return (len + (1 << lg) - 1) >> lg; }
__device__ __forceinline__ Plan make_plan(int64_t n64, int64_t n16, int W) {
  Plan p;
  p.lg = 4 * n64 >= (int64_t)W ? 6 : 4;
  p.T = (int)(p.lg == 6 ? n64 : n16);
  p.W = p.T < W ? p.T : W;
  p.per = p.W ? p.T / p.W : 0;
  p.more = p.T - p.per * p.W;
  return p;
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
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// Warps per CTA: as many as the registers allow.  With eight the kernel waited
// for its own instructions two thirds of the time (two warps per scheduler; 16
// rows of 32768: 181 us a step, 172 with twelve).
__host__ __device__ constexpr int split_warps(int NH) { return NH == 1 ? 12 : 8; }

// SPARE (up to four heads): columns 4..7 are heads 0..3 again, and where the others
// take p, rounded, they take what that left, so the second number costs no matrix
// instruction of its own (attention over 1 x 32768: 24.2 us with one, 23.4 so, 23.0
// without the second number; 32 x 4096 ragged 38.2, 37.7 and 37.3).
template <typename T, int D, int NH, bool SPARE>
__global__ void __launch_bounds__(32 * split_warps(NH), 1) kv8_split_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kWarps = split_warps(NH), kThreads = 32 * kWarps;
  constexpr int J = D / 64;             // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;            // m-tiles of O^T
  constexpr uint32_t SLOT = 64 * D;     // bytes
  constexpr int CPR = D / 16;           // 16-byte chunks per row
  constexpr int RPI = 32 / CPR;         // rows per warp-wide copy
  extern __shared__ __align__(1024) unsigned char ring[];
  constexpr int PT = (kMaxRows + kThreads - 1) / kThreads;
  __shared__ int pre[PT * kThreads + 1];  // units of one head in rows before b
  __shared__ int lens[PT * kThreads];     // tokens of row b
  __shared__ long long red[2][kWarps];
  __shared__ int last_s[kWarps];        // the pair that a warp's range ends in

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const uint32_t none = (uint32_t)a.B >> 31;  // 0, unknown to the compiler
  const uint32_t mask = 0x00ff00ffu + none, bits = 0x64806480u + none;
  pdl_trigger();
  bool waited = !a.early;  // (until then everything is read past L1, which the kernel before may still fill)
  if (waited) pdl_wait();

  // the plan: lengths summed over the rows; one position for all rows needs no sum
  const int KV = a.c.KV;
  const bool even = a.pos.stride == 0;
  Plan plan;
  int nu0 = 0, len0 = 0;  // units of a head and tokens, one position for all
  if (even) {
    len0 = kv8_len(a.pos(0), a.c.S);
    plan = make_plan((int64_t)a.B * KV * units(len0, 6), (int64_t)a.B * KV * units(len0, 4), a.W);
    nu0 = units(len0, plan.lg);
  } else {
    int len[PT];
    long long n64 = 0, n16 = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int b = threadIdx.x * PT + i;
      len[i] = b < a.B ? kv8_len(a.pos(b), a.c.S) : 0;
      n64 += units(len[i], 6);
      n16 += units(len[i], 4);
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
    for (int i = 0; i < PT; ++i) mine += units(len[i], plan.lg);
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
      lens[threadIdx.x * PT + i] = len[i];
      base += units(len[i], plan.lg);
    }
    if (threadIdx.x == kThreads - 1) pre[PT * kThreads] = base;
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
    if constexpr (SPARE)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][i][e] += __shfl_xor_sync(0xffffffffu, o[0][i][e], 2);
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
  const int u0 = plan.begin(wi);

  // ---- the load cursor: next segment at unit `un` of pair (nb, nh) ----
  int nb, nh, un, nu, len;
  int rem = plan.begin(wi + 1) - u0;
  if (even) {
    const int pair = u0 / nu0;
    nb = pair / KV;
    nh = pair - nb * KV;
    un = u0 - pair * nu0;
    nu = nu0;
  } else {
    int lo = 0, hi = a.B - 1;  // the last row with KV pre[row] <= u0 (it is not empty)
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if ((int64_t)pre[m] * KV <= u0) lo = m; else hi = m - 1;
    }
    nb = lo;
    nu = pre[nb + 1] - pre[nb];
    const int v = u0 - pre[nb] * KV;
    nh = v / nu;
    un = v - nh * nu;
  }
  len = even ? len0 : lens[nb];
  auto next_seg = [&](Seg& s) -> bool {
    if (rem <= 0) return false;
    if (un == nu) {  // next pair; rows without tokens have none
      un = 0;
      if (++nh == KV) {
        nh = 0;
        ++nb;
        if (!even) {
          while (pre[nb + 1] == pre[nb]) ++nb;
          nu = pre[nb + 1] - pre[nb];
          len = lens[nb];
        }
      }
    }
    const int t = un << plan.lg;
    s.b = nb;
    s.kvh = nh;
    s.blk = t >> 6;
    s.valid = min(64, len - (s.blk << 6));
    s.s0 = (t & 63) >> 4;
    const int n = plan.lg == 6 ? 1 : min(min(4 - s.s0, nu - un), rem);  // units of this block
    s.s1 = min(s.s0 + (n << (plan.lg - 4)), (s.valid + 15) >> 4);
    un += n;
    rem -= n;
    if (!waited && s.blk == (len - 1) >> 6) {
      pdl_wait();
      waited = true;
    }
    const int64_t o = (int64_t)s.b * a.c.s_sb + (int64_t)s.kvh * a.c.s_sh + s.blk;
    s.sk = __ldcg(a.c.ks + o);
    s.sv = __ldcg(a.c.vs + o);
    return true;
  };

  // the warp's two slots: K and V of a block
  const uint32_t slot_k = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * 2 * SLOT, slot_v = slot_k + SLOT;
  // a lane's place in a copy of RPI rows; for V it takes turns (rows / 2 mod 4 decides)
  const uint32_t put_k = slot_k + slot_off<D, false>(lane / CPR, lane % CPR);
  const uint32_t put_v0 = slot_v + slot_off<D, true>(lane / CPR, lane % CPR);
  const uint32_t put_v1 = slot_v + slot_off<D, true>(RPI + lane / CPR, lane % CPR) - RPI * D;
  auto issue = [&](const Seg& s, bool is_v) {
    const int8_t* src = (is_v ? a.c.vq : a.c.kq) + (int64_t)s.b * a.c.q_sb + (int64_t)s.kvh * a.c.q_sh +
                        (int64_t)s.blk * (64 * D) + lane * 16;
    const bool all = s.s1 - s.s0 == 4;
#pragma unroll
    for (int i = 0; i < 64 / RPI; ++i) {
      const int st = i * RPI / 16;
      if (all || (st >= s.s0 && st < s.s1)) cp_async16((is_v ? (i & 1 ? put_v1 : put_v0) : put_k) + i * RPI * D, src + i * 512);
    }
  };

  auto begin_pair = [&](const Seg& s) {
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int h = SPARE ? r & 3 : 8 * n + r;
      const T* qp = static_cast<const T*>(a.q) + (int64_t)s.b * a.q_sb + ((int64_t)s.kvh * a.g + h) * a.q_sh + 16 * c;
      float f[J][16];
      float mx = 0.f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (h < a.g) v = __ldcg(reinterpret_cast<const uint4*>(qp + 64 * j + 8 * e));
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
  issue(cur, false);
  cp_commit();
  issue(cur, true);
  cp_commit();
  begin_pair(cur);
  while (true) {
    more = next_seg(nxt);
    const bool all = cur.s1 - cur.s0 == 4 && cur.valid == 64;  // a whole block
    cp_wait<1>();  // cur's K
    __syncwarp();

    // ---- S = K Q ----
    float sc[NH][4][4];
    {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][s][e] = 0.f;
        if (all || (s >= cur.s0 && s < cur.s1)) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint4 lo = lds16(slot_k + slot_off<D, false>(16 * s + r, 4 * j + c));
            const uint4 hi = lds16(slot_k + slot_off<D, false>(16 * s + r + 8, 4 * j + c));
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
    if (more) issue(nxt, false);
    cp_commit();

    // ---- the block's softmax; tokens outside [16 s0, valid) do not count ----
    if (!all) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s < cur.s0 || s >= cur.s1 || 16 * s + r + 8 * (e >> 1) >= cur.valid) sc[n][s][e] = -INFINITY;
    }
    uint32_t pf[NH][4][2], pr[NH][SPARE ? 1 : 4][2];  // p in fp16, and what the rounding left, in fp16 too
    float fo[NH][2], fb[NH][2];  // factors of the running and of the block's sums
    bool same = true;            // no maximum moved
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float mb[2] = {-INFINITY, -INFINITY}, f[2], ref[2];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) mb[e & 1] = fmaxf(mb[e & 1], sc[n][s][e]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 4));
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 8));
        mb[k] = fmaxf(mb[k], __shfl_xor_sync(0xffffffffu, mb[k], 16));
        f[k] = qinv[n][k] * cur.sk;  // (not negative, so it keeps the order)
        // (a factor that is not finite, or a score: everything below becomes NaN)
        mb[k] = mb[k] == -INFINITY ? 0.f : __fmul_rn(mb[k], f[k]);
        ref[k] = 14.f - mb[k];
        const float mn = fmaxf(m[n][k], mb[k]);
        fo[n][k] = ex2(m[n][k] - mn);
        fb[n][k] = ex2(mb[k] - mn);
        same &= m[n][k] == mn;
        m[n][k] = mn;
      }
      float lb[2] = {0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = ex2(fmaf(sc[n][s][e], f[e & 1], ref[e & 1]));
          if (!all && sc[n][s][e] == -INFINITY) p[e] = 0.f;  // (a factor of 0 would make it NaN: a block of zero keys)
          lb[e & 1] += p[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // tokens 2c, 2c + 1 of head r, tokens 2c + 8, 2c + 9
          const uint32_t h = pack_h2(p[2 * e], p[2 * e + 1]);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          const uint32_t left = pack_h2(p[2 * e] - f.x, p[2 * e + 1] - f.y);
          pf[n][s][e] = transpose8x8(SPARE && c >= 2 ? left : h);
          if constexpr (!SPARE) pr[n][s][e] = transpose8x8(left);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        l[n][k] = l[n][k] * fo[n][k] + lb[k] * fb[n][k];
        fb[n][k] *= cur.sv;
      }
    }
    same = __all_sync(0xffffffffu, same);

    cp_wait<1>();  // cur's V
    __syncwarp();
    // ---- O = O fo + (V^T P) fb ----
    {
      float ob[NH][MT][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) ob[n][i][e] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (all || (s >= cur.s0 && s < cur.s1)) {
          const int t = 16 * s + 2 * c;
          uint32_t v0[MT / 2], v1[MT / 2], v8[MT / 2], v9[MT / 2];  // 2 MT bytes of four tokens, from d = 2 MT r
          auto load = [&](uint32_t* dst, int row) {
            if constexpr (D == 128) {
              const uint4 x = lds16(slot_v + slot_off<D, true>(row, r));
              dst[0] = x.x; dst[1] = x.y; dst[2] = x.z; dst[3] = x.w;
            } else {
              const uint2 x = lds8(slot_v + slot_off<D, true>(row, r >> 1) + 8 * (r & 1));
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
            const uint32_t a0 = i8_pair_to_h2(v0[w], v1[w], k, mask, bits), a1 = i8_pair_to_h2(v0[w], v1[w], k + 1, mask, bits);
            const uint32_t a2 = i8_pair_to_h2(v8[w], v9[w], k, mask, bits), a3 = i8_pair_to_h2(v8[w], v9[w], k + 1, mask, bits);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              mma_h(ob[n][i], a0, a1, a2, a3, pf[n][s][0], pf[n][s][1]);
              if constexpr (!SPARE) mma_h(ob[n][i], a0, a1, a2, a3, pr[n][s][0], pr[n][s][1]);
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!same) o[n][i][e] *= fo[n][e & 1];
            o[n][i][e] = fmaf(ob[n][i][e], fb[n][e & 1], o[n][i][e]);
          }
    }
    __syncwarp();
    if (more) issue(nxt, true);
    cp_commit();
    if (!more) break;
    if (nxt.b != cur.b || nxt.kvh != cur.kvh) {
      const int64_t at = ((int64_t)wi + (int64_t)cur.b * KV + cur.kvh) * a.g;
      end_pair(a.pacc + at * D, a.pml + at * 2);
      begin_pair(nxt);
    }
    cur = nxt;
  }
  cp_wait<0>();
  last_pair = cur.b * KV + cur.kvh;
  }  // (warps with work)
  if (!waited) pdl_wait();  // (what follows this kernel follows the append too)

  // ---- the last partials of the CTA's warps, joined where they are of one pair ----
  __syncthreads();  // the rings are empty
  float* sacc = reinterpret_cast<float*>(ring);          // [warp][g][D]
  float* sml = sacc + (size_t)kWarps * a.g * D;          // [warp][g][2]
  if (last_pair >= 0) end_pair(sacc + (size_t)warp * a.g * D, sml + warp * a.g * 2);
  if (lane == 0) last_s[warp] = last_pair;
  __syncthreads();
  // runs of warps that end in one pair: a (run, head) per warp, 4 dims per lane
  const int theirs = lane < kWarps ? last_s[lane] : -1;
  const int before = __shfl_up_sync(0xffffffffu, theirs, 1);
  const unsigned heads = __ballot_sync(0xffffffffu, theirs >= 0 && (lane == 0 || before != theirs));
  const int runs = __popc(heads) * a.g;
  for (int i = warp; i < runs; i += kWarps) {
    const int run = i / a.g, h = i - run * a.g;
    unsigned rest = heads;
    for (int k = 0; k < run; ++k) rest &= rest - 1;
    const int w0 = __ffs(rest) - 1, pair = last_s[w0];
    rest &= rest - 1;
    int w1 = rest ? __ffs(rest) - 1 : kWarps;
    while (last_s[w1 - 1] != pair) --w1;  // (warps without work)
    // lane = warp: its max and sum
    const bool in = lane >= w0 && lane < w1;
    const float2 ml = in ? *reinterpret_cast<const float2*>(sml + (lane * a.g + h) * 2) : make_float2(-INFINITY, 0.f);
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float f = in ? ex2(ml.x - mx) : 0.f;
    const float sum = warp_sum(in ? ml.y * f : 0.f);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = w0; q < w1; ++q) {
      const float fq = __shfl_sync(0xffffffffu, f, q);
      if (4 * lane < D) {
        const float4 o4 = *reinterpret_cast<const float4*>(sacc + ((size_t)q * a.g + h) * D + 4 * lane);
        v.x = fmaf(o4.x, fq, v.x); v.y = fmaf(o4.y, fq, v.y); v.z = fmaf(o4.z, fq, v.z); v.w = fmaf(o4.w, fq, v.w);
      }
    }
    const int64_t at = ((int64_t)blockIdx.x * kWarps + w0 + pair) * a.g + h;
    if (4 * lane < D) *reinterpret_cast<float4*>(a.pacc + at * D + 4 * lane) = v;
    if (lane == 0) *reinterpret_cast<float2*>(a.pml + at * 2) = make_float2(mx, sum);
  }
}

// ---------------------------------------------------------------------------
// join: out[b, h] = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k over the
// partials of the pair.  A warp per head, lane = 4 dims; a few partials each, so
// no more threads, and nothing to wait for among them (with a CTA per pair 32 x
// 4096 ragged took 38 us instead of 36, both kernels).
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 4;

template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) kv8_join_kernel(const __grid_constant__ AttnArgs a) {
  const int lane = threadIdx.x & 31, D = a.c.D, KV = a.c.KV;
  const int b = blockIdx.y, h = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (h >= a.H) return;
  const int kvh = h / a.g, hl = h - kvh * a.g;
  const int len = kv8_len(a.pos(b), a.c.S);
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + 4 * lane;
  const bool mine = 4 * lane < D;
  if (len == 0) {  // a row that is not there
    if (mine)
      for (int e = 0; e < 4; ++e) out[e] = from_f<T>(0.f);
    return;
  }
  long long s[4];  // units of 64 and of 16 tokens, over all rows and over the rows before b
  if (a.pos.stride == 0) {
    s[0] = (long long)a.B * units(len, 6);
    s[1] = (long long)a.B * units(len, 4);
    s[2] = (long long)b * units(len, 6);
    s[3] = (long long)b * units(len, 4);
  } else {
    s[0] = s[1] = s[2] = s[3] = 0;
    for (int i = lane; i < a.B; i += 32) {
      const int n = kv8_len(a.pos(i), a.c.S), n64 = units(n, 6), n16 = units(n, 4);
      s[0] += n64;
      s[1] += n16;
      if (i < b) {
        s[2] += n64;
        s[3] += n16;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
  }
  const Plan plan = make_plan(s[0] * KV, s[1] * KV, a.W);
  const int nu = units(len, plan.lg);
  const int lo = (int)(plan.lg == 6 ? s[2] : s[3]) * KV + kvh * nu, hi = lo + nu;
  const int i0 = plan.warp_of(lo), i1 = plan.warp_of(hi - 1);
  const int64_t p = (int64_t)b * KV + kvh;
  // partials: warp i0's, the first of each later CTA, and warp i1's if it goes on to the next pair
  // (otherwise it ends here, as all between do, and is joined to its CTA's)
  const int first = (i0 / a.cw + 1) * a.cw;
  const int later = i1 < first ? 0 : (i1 - first) / a.cw + 1;
  const bool own = i1 > i0 && i1 % a.cw != 0 && plan.begin(i1 + 1) > hi;
  const int n = 1 + later + (own ? 1 : 0);
  // slot of partial k, from the pair's first: warps apart
  const int64_t slot0 = (i0 + p) * a.g + hl;
  auto off_of = [&](int k) { return (k == 0 ? 0 : k <= later ? first + (k - 1) * a.cw - i0 : i1 - i0) * a.g; };
  const float* pml = a.pml + slot0 * 2;
  const float* pacc = a.pacc + slot0 * D + 4 * lane;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 16;  // partials at a time: their loads go out together
  for (int k0 = 0; k0 < n; k0 += U) {
    const float2 ml = lane < U && k0 + lane < n ? *reinterpret_cast<const float2*>(pml + off_of(k0 + lane) * 2)
                                                : make_float2(-INFINITY, 0.f);
    float4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (mine && k0 + k < n) v[k] = *reinterpret_cast<const float4*>(pacc + off_of(k0 + k) * D);
    }
    float mn = ml.x;
#pragma unroll
    for (int o = U / 2; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mn = fmaxf(__shfl_sync(0xffffffffu, mn, 0), m);
    const float f0 = ex2(m - mn), f = ex2(ml.x - mn);
    m = mn;
    l = l * f0 + warp_sum(ml.y * f);
    acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float fk = __shfl_sync(0xffffffffu, f, k);
      acc.x = fmaf(v[k].x, fk, acc.x); acc.y = fmaf(v[k].y, fk, acc.y);
      acc.z = fmaf(v[k].z, fk, acc.z); acc.w = fmaf(v[k].w, fk, acc.w);
    }
  }
  if (mine) {
    const float inv = 1.f / l;
    out[0] = from_f<T>(acc.x * inv);
    out[1] = from_f<T>(acc.y * inv);
    out[2] = from_f<T>(acc.z * inv);
    out[3] = from_f<T>(acc.w * inv);
  }
}

// ---------------------------------------------------------------------------
// any shape: one CTA per (head, row), a warp per token, D <= 256.  For types and
// dims that no served model of this package has; nothing is shared between the
// heads of a group, so it reads the cache g times (from L2).
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kGenericThreads) kv8_generic_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int E = 8;  // dims per lane
  __shared__ float acc_s[kGenericWarps][256];
  __shared__ float m_s[kGenericWarps], l_s[kGenericWarps];
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
  for (int64_t t = warp; t < len; t += kGenericWarps) {
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
    for (int w = 1; w < kGenericWarps; ++w) mm = fmaxf(mm, m_s[w]);
    float num = 0.f, den = 0.f;
    for (int w = 0; w < kGenericWarps; ++w) {
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

int cta_warps(const b200mm_kv8& c, int H) { return split_warps(H / c.KV <= 8 ? 1 : 2); }
// CTAs of the split kernel: one per SM, fewer where the capacity has no work for them
int split_ctas(const b200mm_kv8& c, int rows, int cw) {
  const int64_t most = (int64_t)rows * c.KV * ((c.S + 15) / 16);
  const int64_t need = (most + cw - 1) / cw;
  const int sms = num_sms(current_device());
  return (int)(need < sms ? need : sms);
}

template <typename T, int D, int NH, bool SPARE>
int run_fast(const AttnArgs& a, cudaStream_t st) {
  constexpr size_t smem = (size_t)split_warps(NH) * 2 * 64 * D;
  auto kern = kv8_split_kernel<T, D, NH, SPARE>;
  const int dev = current_device();
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64) return B200MM_ERR_DEVICE;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return B200MM_ERR_LAUNCH;
    configured[dev] = true;
  }
  cudaError_t e = launch_pdl(kern, dim3(a.W / a.cw), dim3(32 * a.cw), smem, st, a);
  if (e != cudaSuccess) return B200MM_ERR_LAUNCH;
  e = launch_pdl(kv8_join_kernel<T>, dim3((a.H + kJoinWarps - 1) / kJoinWarps, a.B), dim3(32 * kJoinWarps), 0, st, a);
  return e == cudaSuccess ? B200MM_OK : B200MM_ERR_LAUNCH;
}

template <typename T>
int run(const AttnArgs& a, bool fast, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (fast) {
      if (a.c.D == 128)
        return a.g <= 4 ? run_fast<T, 128, 1, true>(a, st)
               : a.g <= 8 ? run_fast<T, 128, 1, false>(a, st) : run_fast<T, 128, 2, false>(a, st);
      return a.g <= 4 ? run_fast<T, 64, 1, true>(a, st)
             : a.g <= 8 ? run_fast<T, 64, 1, false>(a, st) : run_fast<T, 64, 2, false>(a, st);
    }
  }
  return launch_pdl(kv8_generic_kernel<T>, dim3(a.H, a.B), dim3(kGenericThreads), 0, st, a) == cudaSuccess
             ? B200MM_OK
             : B200MM_ERR_LAUNCH;
}

}  // namespace

size_t kv8_decode_workspace_bytes(const b200mm_kv8& c, int B, int H) {
  if (!fast_shape(c, H)) return 0;
  const int rows = B < kMaxRows ? B : kMaxRows;
  const int cw = cta_warps(c, H);
  const size_t slots = (size_t)split_ctas(c, rows, cw) * cw + (size_t)rows * c.KV;
  return slots * (H / c.KV) * (c.D + 2) * sizeof(float);
}

int kv8_decode(const b200mm_kv8& c, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
               int B, int H, Kv8Pos pos, float scale, void* ws, bool early, cudaStream_t st) {
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
    a.early = early && b0 == 0;  // (a later launch follows the one before, with the same workspace)
    if (fast) {
      a.cw = cta_warps(c, H);
      a.W = split_ctas(c, a.B, a.cw) * a.cw;
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
