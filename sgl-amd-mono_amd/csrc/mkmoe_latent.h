// What the latent attention's sources share: a cache row's parts, conversions, the matrix instruction,
// loads into LDS with the waits that they need, and the checks of arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "../../include/mkmoe.h"
#include "mkmoe_numerics.h"

namespace mkmoe_latent {

using mkmoe::bf2f;
using mkmoe::f2u;
using mkmoe::u2f;

constexpr int kL = MKMOE_LATENT_DIM;    // 512
constexpr int kR = MKMOE_LATENT_ROPE;   // 64
constexpr int kRow = kL + kR;           // values a cache row
constexpr int kMxScales = kL / 32;
constexpr int kMxRow = MKMOE_LATENT_MX_ROW;
constexpr int kNope = MKMOE_LATENT_NOPE, kV = MKMOE_LATENT_V;
static_assert(kMxRow == kL + kMxScales + 2 * kR && kMxRow % 16 == 0, "MXFP8 rows in whole 16-byte pieces");

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define MKMOE_LDS __attribute__((address_space(3)))

__device__ __forceinline__ float bf_lo(uint32_t w) { return u2f(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return u2f(w & 0xffff0000u); }
// two fp32 as bf16 (nearest even, NaN kept), a in the low half
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// 8 e4m3 codes (bytes of w0 then w1) times s, a power of two, as bf16: exact
__device__ __forceinline__ u32x4 fp8x8(uint32_t w0, uint32_t w1, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
  return u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
               __builtin_bit_cast(uint32_t, d)};
}
__device__ __forceinline__ float e8m0(uint32_t e) { return u2f(e << 23); }

// the first error of a call since the last clear: a page, slot, position, length or query range
// outside its bounds, and the token or sequence that had it
__device__ inline void record(int32_t* err, int code, int where) {
  if (atomicCAS(err + MKMOE_LATENT_ERRW_CODE, 0, code) == 0) err[MKMOE_LATENT_ERRW_WHERE] = where;
  atomicAdd(err + MKMOE_LATENT_ERRW_COUNT, 1);
}

// Bytes from global memory straight into LDS: lane l's land at lds + 16 l (4 l). One asm
// statement, so that the compiler does not wait for it before other reads of LDS; the caller
// waits (wait_loads) before the bytes are read. M0 may be read one wait state after it was written,
// which the statement holds too
__device__ __forceinline__ void lds_dma16(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds) : "memory", "m0");
}
// (lane l's from base + at. A base that a VALU instruction wrote, v_readlane or the reload of a spilled one,
// may be read 5 wait states later: the compiler does not see the load, so the statement holds them)
__device__ __forceinline__ void lds_dma16(const void* base, uint32_t at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(base), "s"(lds)
               : "memory", "m0");
}
// waits until at most N of the wave's loads are on their way (they complete in order)
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// the same for all of them, as the compiler's own wait: it would otherwise place a wait for the
// registers that page entries or queries went to in the tile loop, which counts the tiles' loads too
__device__ __forceinline__ void wait_all() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0, expcnt 7 (none), lgkmcnt 15 (none)
  asm volatile("" ::: "memory");
}
// every wave's LDS accesses before it are done, and loads stay on their way across it
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// LDS at a byte offset
template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(MKMOE_LDS const T*)(uintptr_t)at;
}

// ---------------------------------------------------------------- host
inline bool aligned(const void* q, size_t a) { return ((uintptr_t)q % a) == 0; }
inline bool strides8(int64_t a, int64_t b) { return a >= 0 && b >= 0 && a % 8 == 0 && b % 8 == 0; }
// no two rows of an output share a place
inline bool rows_apart(int64_t ts, int64_t tokens, int64_t hs, int64_t heads, int64_t width) {
  const bool by_token = ts >= hs;
  const int64_t big = by_token ? ts : hs, n_big = by_token ? tokens : heads;
  const int64_t small = by_token ? hs : ts, n_small = by_token ? heads : tokens;
  if (n_small <= 1) return n_big <= 1 || big >= width;
  return small >= width && (n_big <= 1 || (big - width) / small >= n_small - 1);
}

inline int check_cache(const mkmoe_latent_cache& c) {
  if (!c.data) return MKMOE_ERR_NULL;
  if (!aligned(c.data, 16)) return MKMOE_ERR_ALIGN;
  if (c.fmt != MKMOE_LATENT_BF16 && c.fmt != MKMOE_LATENT_MXFP8) return MKMOE_ERR_ARG;
  if (c.page_size < 1 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)) != 0) return MKMOE_ERR_ARG;
  if (c.pages < 1 || c.pages > (int64_t)0x7fffffff / c.page_size) return MKMOE_ERR_ARG;
  return MKMOE_OK;
}
// mkmoe_latent_append (its checks, then its launch) for rows that are attended with next: the query of a token
// that cannot be stored becomes NaN
int append_for_step(const mkmoe_latent_append_io* io, void* ws, size_t ws_bytes, hipStream_t st);
inline int launched() { return hipGetLastError() == hipSuccess ? MKMOE_OK : MKMOE_ERR_LAUNCH; }

}  // namespace mkmoe_latent
