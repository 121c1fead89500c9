// What the decode kernels (attention.hip), the prefill kernels
// (attention_prefill.hip) and the paged ones (paged.hip) of the attention share.
#pragma once
#include "common.h"

namespace htn {

constexpr int D = HTN_HEAD_DIM;
constexpr int kSplit = 64;  // cache slots per tile

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the four quads'
// copies of one query row): gfx950's row-swap permutes, no LDS round trip.
// permlane16_swap pairs row r with row r ^ 1 and permlane32_swap the wave's
// halves; both results of each swap hold the two partners.
__device__ __forceinline__ float quad_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float quad_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Operand reads of the staged tiles of the prefill and paged kernels (LDS-direct data, read
// by inline asm: the compiler would wait for every load in flight before an
// ordinary LDS read of such a buffer), issued without their waits: issue, run
// other work, then a wait that names the registers as operands so no use of
// them moves above it. K: one 32-dim step for the four 16-slot M-tiles of a
// 64-slot tile; V^T: transpose reads as attention.hip's read_vt_tr.
template <int OFF>
__device__ __forceinline__ void issue_k_pf(uint32_t addr, u32x4 (&k)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%5\n\t"
      "ds_read_b128 %1, %4 offset:%6\n\t"
      "ds_read_b128 %2, %4 offset:%7\n\t"
      "ds_read_b128 %3, %4 offset:%8"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3])
      : "v"(addr), "n"(OFF), "n"(OFF + 4096), "n"(OFF + 8192), "n"(OFF + 12288)
      : "memory");
}

typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

template <int OFF>
__device__ __forceinline__ void issue_vt_tr(const uint32_t (&va)[8], u32x2_t (&w)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%16\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%16\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
      "ds_read_b64_tr_b16 %4, %12 offset:%16\n\t"
      "ds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
      "ds_read_b64_tr_b16 %6, %14 offset:%16\n\t"
      "ds_read_b64_tr_b16 %7, %15 offset:%16"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]),
        "=&v"(w[6]), "=&v"(w[7])
      : "v"(va[0]), "v"(va[1]), "v"(va[2]), "v"(va[3]), "v"(va[4]), "v"(va[5]), "v"(va[6]),
        "v"(va[7]), "n"(OFF)
      : "memory");
}

__device__ __forceinline__ void wait_k16(u32x4 (&k)[4][4]) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(k[0][0]), "+v"(k[0][1]), "+v"(k[0][2]), "+v"(k[0][3]), "+v"(k[1][0]),
                 "+v"(k[1][1]), "+v"(k[1][2]), "+v"(k[1][3]), "+v"(k[2][0]), "+v"(k[2][1]),
                 "+v"(k[2][2]), "+v"(k[2][3]), "+v"(k[3][0]), "+v"(k[3][1]), "+v"(k[3][2]),
                 "+v"(k[3][3])
               :
               : "memory");
}

__device__ __forceinline__ void wait_v32(u32x2_t (&w)[4][8]) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(w[0][0]), "+v"(w[0][1]), "+v"(w[0][2]), "+v"(w[0][3]), "+v"(w[0][4]),
                 "+v"(w[0][5]), "+v"(w[0][6]), "+v"(w[0][7]), "+v"(w[1][0]), "+v"(w[1][1]),
                 "+v"(w[1][2]), "+v"(w[1][3]), "+v"(w[1][4]), "+v"(w[1][5]), "+v"(w[1][6]),
                 "+v"(w[1][7]), "+v"(w[2][0]), "+v"(w[2][1]), "+v"(w[2][2]), "+v"(w[2][3]),
                 "+v"(w[2][4]), "+v"(w[2][5]), "+v"(w[2][6]), "+v"(w[2][7]), "+v"(w[3][0]),
                 "+v"(w[3][1]), "+v"(w[3][2]), "+v"(w[3][3]), "+v"(w[3][4]), "+v"(w[3][5]),
                 "+v"(w[3][6]), "+v"(w[3][7])
               :
               : "memory");
}

__device__ __forceinline__ void wait_v16(u32x2_t (&w)[2][8]) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(w[0][0]), "+v"(w[0][1]), "+v"(w[0][2]), "+v"(w[0][3]), "+v"(w[0][4]),
                 "+v"(w[0][5]), "+v"(w[0][6]), "+v"(w[0][7]), "+v"(w[1][0]), "+v"(w[1][1]),
                 "+v"(w[1][2]), "+v"(w[1][3]), "+v"(w[1][4]), "+v"(w[1][5]), "+v"(w[1][6]),
                 "+v"(w[1][7])
               :
               : "memory");
}

// Causal attention over many queries per sequence, without a split.
struct PrefillArgs {
  const bf16_t* q; long q_sb, q_sh, q_st;
  const bf16_t* keys; const bf16_t* values; long cap;
  const int64_t* pos;
  bf16_t* out;  // row (b, h, t) at b*o_sb + h*o_sh + t*o_st (dims contiguous)
  long o_sb, o_sh, o_st;
  int B, Hq, Hkv, G, Q;
  int turn;     // attention_prefill_long: the query rank from which ranks run in reverse
  float scale;
};

// Needs 16-byte query fragments and 8-byte output stores; one launch, no scratch.
int prefill_attention(PrefillArgs& a, hipStream_t st);

}  // namespace htn
