// 8-bit KV cache: layout, bounds and launch entries shared by kv8.cu (append,
// expand) and kv8_attn.cu (decode attention).
#pragma once
#include <cstddef>

#include "common.cuh"

// the layout that the Python mirror of the struct has
static_assert(sizeof(b200mm_kv8) == 120 && offsetof(b200mm_kv8, S) == 96 && offsetof(b200mm_kv8, KV) == 104);

namespace b200mm {

constexpr int kKv8Block = 64;  // tokens that share a scale (per row, head, and K / V)

// Positions of a call's rows: one on the host for every row, or on the device
// one for all (stride 0) or one for each row (stride 1).
struct Kv8Pos {
  const int64_t* dev;
  int64_t host;
  int stride;
  __device__ __forceinline__ int64_t operator()(int b) const { return dev ? __ldcg(dev + (int64_t)b * stride) : host; }
};

// Tokens that row b attends to, for its last position p: p + 1, at most the capacity; none below 0.
__device__ __forceinline__ int kv8_len(int64_t p, int64_t S) { return p < 0 ? 0 : (int)(p < S ? p + 1 : S); }

// int8 bytes i of two words -> fp16x2 (exact): the bytes, sign-flipped, become
// the low mantissa bits of 1024 + (q + 128), and subtracting 1152 leaves q.
// `mask` is 0x00ff00ff and `bits` 0x64806480, in registers: one logic
// instruction takes one literal.
__device__ __forceinline__ uint32_t i8_pair_to_h2(uint32_t w0, uint32_t w1, int i, uint32_t mask, uint32_t bits) {
  const uint32_t x = __byte_perm(w0, w1, (uint32_t)(0x4400 + 0x1111 * i));
  uint32_t h;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(h) : "r"(x), "r"(mask), "r"(bits));  // (x & mask) ^ bits
  const __half2 v =
      __hsub2(*reinterpret_cast<const __half2*>(&h), __half2(__float2half(1152.f), __float2half(1152.f)));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// `late`, `early`: a decode step's two halves.  The append lets the attention start as soon as all
// before the step is done; the attention waits for the append only where it comes to the last block
// of a row, which is all that the append of one token changes.
int kv8_append(const b200mm_kv8& c, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void* v,
               int64_t v_sb, int64_t v_sh, int64_t v_st, int B, int64_t T, Kv8Pos pos, bool late, cudaStream_t st);
int kv8_expand(const b200mm_kv8& c, void* k, void* v, int64_t o_sb, int64_t o_sh, int64_t o_st, int B, int64_t L,
               cudaStream_t st);
size_t kv8_decode_workspace_bytes(const b200mm_kv8& c, int B, int H);
int kv8_decode(const b200mm_kv8& c, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
               int B, int H, Kv8Pos pos, float scale, void* ws, bool early, cudaStream_t st);

}  // namespace b200mm
