// Latent attention of a decode step on gfx950 (MI355X): HIP kernels and the C ABI of the latent
// section of include/mkmoe.h.
//
// A token's keys and values are one shared row: 512 latent values c (RMS-normed) and 64 rotated
// rope values k_pe, in a paged cache, as bf16 (1152 bytes) or MXFP8 (512 e4m3 codes, 16 E8M0
// scales, 64 bf16 rope values: 656 bytes). In the absorbed form every head's query is 512 + 64
// values against that row, and the row's latent part is the value too:
//   s = scale (q_lat . c + q_pe . k_pe),  o = sum softmax(s) c.
//
//   k_latent_append   norm, rotate and write a step's rows; rotate the query's rope part
//   k_latent_rows     the values that cache rows stand for
//   k_latent_attend   the absorbed attention, its work cut into equal shares over the card
//   k_latent_merge    joins the shares of a sequence that was cut
//   k_latent_absorb / k_latent_expand   the two products of every head with its weights
//   k_latent_front    a step's append and absorb in one launch
//
// Times below are of an MI355X, in graph replays. It copies 5.19 TB/s and multiplies bf16 matrices
// at 1.25 PFLOP/s, which make the floors.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <type_traits>

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
__device__ void record(int32_t* err, int code, int where) {
  if (atomicCAS(err + MKMOE_LATENT_ERRW_CODE, 0, code) == 0) err[MKMOE_LATENT_ERRW_WHERE] = where;
  atomicAdd(err + MKMOE_LATENT_ERRW_COUNT, 1);
}

// ---------------------------------------------------------------- append
struct AppendParams {
  const uint16_t* kv;
  const uint16_t* norm_w;
  const float* cos_sin;
  const void* positions;
  const void* slots;
  const uint16_t* q;
  uint16_t* q_out;
  uint8_t* cache;
  int32_t* err;
  int64_t kv_stride, q_ts, q_hs, o_ts, o_hs;
  int64_t rows, table_rows;
  int tokens, heads, half, wide, kv_blocks, mark;
  float eps;
};

__device__ __forceinline__ int64_t index_at(const void* p, int i, int wide) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// the lane's 8 values (16 bytes at value 8 j of a 64-value row, j = lane % 8) rotated by the
// row's angles: pairs (2 i, 2 i + 1), or (i, i + 32) with the partner's values 4 lanes away
__device__ __forceinline__ u32x4 rotate8(u32x4 v, const float* cs, int j, int half) {
  float x[8];
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf_lo(w[i]);
    x[2 * i + 1] = bf_hi(w[i]);
  }
  uint32_t o[4];
  if (!half) {
    const f32x4 c = *(const f32x4*)(cs + 4 * j), s = *(const f32x4*)(cs + kR / 2 + 4 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = pack_bf(x[2 * i] * c[i] - x[2 * i + 1] * s[i], x[2 * i + 1] * c[i] + x[2 * i] * s[i]);
  } else {
    const int jj = j & 3;
    const f32x4 c0 = *(const f32x4*)(cs + 8 * jj), c1 = *(const f32x4*)(cs + 8 * jj + 4);
    const f32x4 s0 = *(const f32x4*)(cs + kR / 2 + 8 * jj), s1 = *(const f32x4*)(cs + kR / 2 + 8 * jj + 4);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor(x[i], 4, 64);
      const float c = i < 4 ? c0[i & 3] : c1[i & 3], s = i < 4 ? s0[i & 3] : s1[i & 3];
      y[i] = j < 4 ? x[i] * c - other * s : x[i] * c + other * s;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack_bf(y[2 * i], y[2 * i + 1]);
  }
  return u32x4{o[0], o[1], o[2], o[3]};
}

// fp32 that a later rounding to fewer bits takes to the place where it would take x: cut off, the last
// bit set where something was
__device__ __forceinline__ float to_odd(double x) {
  float f = __double2float_rz(x);
  if ((double)f != x && fabsf(f) < INFINITY) f = u2f(f2u(f) | 1u);
  return f;
}

// A wave a token of the first kv_blocks workgroups: lane l holds latent values 8 l .. 8 l + 7,
// lanes 0 .. 7 the rope values too. The other workgroups rotate the query, 8 lanes a head's 64 values.
// Each value is read and written once: bound by memory on a prompt (8191 rows of 32 heads, 88 MB:
// 17.4 us in graph replays, 5.1 TB/s) and by one trip to it on a decode step (7 rows 2.8 us). The
// norm's sum is formed in 64 bits, and so are MXFP8's products: a code next to a border is the one that
// the definition has (fp32 missed one in some 10^5 of them).
// STEP: the query rows are attended with next, so that those of a token that cannot be stored become NaN
template <bool MX, bool STEP>
__device__ __forceinline__ void append_block(const AppendParams& p, int block) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (block < p.kv_blocks) {
    const int t = block * 4 + wave;
    if (t >= p.tokens) return;
    const int64_t slot = index_at(p.slots, t, p.wide), pos = index_at(p.positions, t, p.wide);
    if (slot < 0) return;  // a padded row
    if (slot >= p.rows || pos < 0 || pos >= p.table_rows) {
      if (lane == 0) record(p.err, slot >= p.rows ? MKMOE_LATENT_ERR_SLOT : MKMOE_LATENT_ERR_POSITION, t);
      return;
    }
    const uint16_t* src = p.kv + (int64_t)t * p.kv_stride;
    uint8_t* dst = p.cache + slot * (MX ? kMxRow : 2 * kRow);
    const u32x4 v = *(const u32x4*)(src + 8 * lane);
    u32x4 pe = {0, 0, 0, 0};
    if (lane < 8) pe = *(const u32x4*)(src + kL + 8 * lane);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = bf_lo(w[i]);
      y[2 * i + 1] = bf_hi(w[i]);
    }
    if (p.norm_w) {
      const u32x4 nv = *(const u32x4*)(p.norm_w + 8 * lane);
      const uint32_t nw[4] = {nv.x, nv.y, nv.z, nv.w};
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += (double)y[i] * (double)y[i];
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) ss += __shfl_xor(ss, d, 64);
      const double rstd = 1.0 / sqrt(ss / kL + (double)p.eps);
      // (without eps, rows of bf16's subnormals: rstd reaches 2^138, past fp32. Its power of two goes to the values)
      const bool far = rstd > 0x1p100;
      const float up = far ? 0x1p64f : 1.0f, r32 = (float)(far ? rstd * 0x1p-64 : rstd);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (MX) {
          y[2 * i] = to_odd((double)y[2 * i] * rstd * (double)bf_lo(nw[i]));
          y[2 * i + 1] = to_odd((double)y[2 * i + 1] * rstd * (double)bf_hi(nw[i]));
        } else {
          y[2 * i] = y[2 * i] * up * r32 * bf_lo(nw[i]);
          y[2 * i + 1] = y[2 * i + 1] * up * r32 * bf_hi(nw[i]);
        }
      }
    }
    if constexpr (MX) {
      // 32 values are 4 lanes; the scale is the least power of two that keeps them within 448
      // (as the block's own MXFP8 activations have it), so no code saturates; codes straight from the values
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(y[i]));
      top = fmaxf(top, __shfl_xor(top, 1, 64));
      top = fmaxf(top, __shfl_xor(top, 2, 64));
      const int e = mkmoe::vllm_code(top);
      const float inv = mkmoe::mx_inv(e);
      int w0 = 0, w1 = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // (NaN passes both comparisons)
        const float q = y[i] * inv;
        y[i] = q > 448.0f ? 448.0f : (q < -448.0f ? -448.0f : q);
      }
      w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w0, false);
      w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
      w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], w1, false);
      w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
      *(u32x2*)(dst + 8 * lane) = u32x2{(uint32_t)w0, (uint32_t)w1};
      if ((lane & 3) == 0) dst[kL + (lane >> 2)] = (uint8_t)e;
    } else {
      *(u32x4*)(dst + 16 * lane) = u32x4{pack_bf(y[0], y[1]), pack_bf(y[2], y[3]), pack_bf(y[4], y[5]), pack_bf(y[6], y[7])};
    }
    if (lane < 8) {
      const u32x4 o = rotate8(pe, p.cos_sin + pos * kR, lane, p.half);
      *(u32x4*)(dst + (MX ? kL + kMxScales : 2 * kL) + 16 * lane) = o;
    }
    return;
  }
  const int64_t r = ((int64_t)(block - p.kv_blocks) * 4 + wave) * 8 + (lane >> 3);
  if (r >= (int64_t)p.tokens * p.heads) return;
  const int t = (int)(r / p.heads), h = (int)(r - (int64_t)t * p.heads), j = lane & 7;
  const int64_t pos = index_at(p.positions, t, p.wide);
  const bool lost = pos < 0 || pos >= p.table_rows, unstored = STEP && index_at(p.slots, t, p.wide) >= p.rows;
  u32x4* to = (u32x4*)(p.q_out + t * p.o_ts + h * p.o_hs + 8 * j);
  if (lost || unstored) {
    const bool padded = index_at(p.slots, t, p.wide) < 0;  // it needs no position
    if (lost && !padded && j == 0 && h == 0) record(p.err, MKMOE_LATENT_ERR_POSITION, t);
    const uint32_t v = padded ? 0 : 0x7fc07fc0u;
    if (padded || STEP || p.mark) *to = u32x4{v, v, v, v};
    return;
  }
  const u32x4 v = *(const u32x4*)(p.q + t * p.q_ts + h * p.q_hs + 8 * j);
  *to = rotate8(v, p.cos_sin + pos * kR, j, p.half);
}

template <bool MX>
__global__ __launch_bounds__(256) void k_latent_append(AppendParams p) {
  append_block<MX, false>(p, blockIdx.x);
}

// ---------------------------------------------------------------- rows as values
struct RowsParams {
  const uint8_t* cache;
  const void* slots;
  uint16_t* out;
  int32_t* err;
  int64_t rows;
  int tokens, wide;
};

// a wave a row: lane l writes the latent values 8 l .. 8 l + 7, lanes 0 .. 7 the rope values
template <bool MX>
__global__ __launch_bounds__(256) void k_latent_rows(RowsParams p) {
  const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.tokens) return;
  const int64_t slot = index_at(p.slots, t, p.wide);
  u32x4 c = {0, 0, 0, 0}, pe = {0, 0, 0, 0};
  if (slot >= p.rows) {
    if (lane == 0) record(p.err, MKMOE_LATENT_ERR_SLOT, t);
  } else if (slot >= 0) {
    const uint8_t* src = p.cache + slot * (MX ? kMxRow : 2 * kRow);
    if constexpr (MX) {
      const u32x2 q = *(const u32x2*)(src + 8 * lane);
      c = fp8x8(q.x, q.y, e8m0(src[kL + (lane >> 2)]));
    } else {
      c = *(const u32x4*)(src + 16 * lane);
    }
    if (lane < 8) pe = *(const u32x4*)(src + (MX ? kL + kMxScales : 2 * kL) + 16 * lane);
  }
  uint16_t* dst = p.out + (int64_t)t * kRow;
  *(u32x4*)(dst + 8 * lane) = c;
  if (lane < 8) *(u32x4*)(dst + kL + 8 * lane) = pe;
}

// ---------------------------------------------------------------- attend
constexpr int kN = 32;          // cached tokens a tile
constexpr int kShares = 256;    // equal shares of the work, a workgroup each: one a CU
constexpr int kThreads = 512;   // 8 waves
constexpr int kMaxSeqs = MKMOE_LATENT_MAX_SEQS;
constexpr int kRowsMax = 64;    // query rows a row tile holds at most
constexpr int kPStride = kN + 16;  // bf16 of a row of P: 96 bytes, whose 16-byte reads meet every bank once
constexpr int kTileBytes = kN * kRow * 2;  // a tile's rows in LDS, bf16: the latent parts, then the rope parts
constexpr int kRopeAt = kN * kL * 2;
constexpr int kRing = 4;        // bf16 cache: tiles in LDS, one in use and three on their way
constexpr int kMxRing = 3;      // MXFP8: raw tiles on their way
constexpr int kSetup = 8;       // see setup()
constexpr int kNarrow = 4096;   // see k_latent_attend
constexpr int kEnts = 4;        // tiles whose page entries are in LDS
// A row's maximum is moved only where a score passes it by more than 2^kSlack: numerators then stay
// below 2^kSlack (bf16 and fp32 keep their relative precision there). After the first tiles almost
// none does, so that the waves need not agree on a tile's maxima before its numerators, nor rescale
constexpr float kSlack = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

// bf16 parts that a numerator is taken as, a matrix operand: two leave out 2^-17 of it, one 2^-9. The second one's
// products fit under the tile's loads at 32 rows of a bf16 cache (48 sequences of 8192 102 to 105 us either way, 36
// ragged ones 46 and 45; error of the outputs 0.0021 -> 0.0017, which is their own rounding). At 64 rows the MFMAs
// and LDS bound the tile, and in MXFP8 the waves that multiply unpack as well (64 sequences 105 us, with two parts
// 115; 48 of 16384 141 and 156)
template <int M, bool MX>
constexpr int kPParts = M == 32 && !MX ? 2 : 1;

// what the end of a share cut, for the merge: the row tile that goes on in the next share
struct Cut {
  int32_t parts;        // 0: nothing was cut there
  int32_t share;        // the first share with a part of it, in slot 2 share + 1; the others are in
                        // slots 2 (share + 1), 2 (share + 2) ..
  int32_t t0, r0, nrows;  // the sequence's first query token, the tile's rows of it
  int32_t base;         // tokens that its first query sees (may be negative)
  int32_t m;            // rows a tile: 32 or 64
  int32_t unused;
};

struct AttendParams {
  const uint16_t* ql;
  const uint16_t* qp;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;  // NULL: n query tokens a sequence
  void* out;  // bf16, or fp32 (f32)
  float* lse;
  int32_t* err;
  int32_t* covered;  // [2]: receives the rows that the sequences have by starts, from and up to
  Cut* cut;        // [kShares]
  float* part_o;   // [2 kShares][M][512]
  float* part_ml;  // [2 kShares][M][2]
  int64_t ql_ts, ql_hs, qp_ts, qp_hs, o_ts, o_hs;
  int64_t table_stride;
  int pages, seqs, tokens, heads, n, max_len, page_shift, f32;
  uint32_t per_head;  // 2^32 / heads, rounded up
  float scale2;       // scale log2(e)
};

// four attended values, rounded where the caller takes bf16
__device__ __forceinline__ void store4(const AttendParams& p, int64_t to, f32x4 v) {
  if (p.f32)
    *(f32x4*)((float*)p.out + to) = v;
  else
    *(u32x2*)((uint16_t*)p.out + to) = u32x2{pack_bf(v[0], v[1]), pack_bf(v[2], v[3])};
}

// a query row's token: exact for rows below 2^24 and up to 128 heads (the product is off by less
// than rows x heads <= 2^31 of 2^32)
__device__ __forceinline__ int over_heads(const AttendParams& p, int row) {
  return p.heads == 1 ? row : (int)__umulhi((uint32_t)row, p.per_head);
}

// a sequence's query tokens and length, clamped to their bounds
struct Seq {
  int t0, n, len;
  bool bad, back;  // outside its bounds; its query starts run backwards
};
__device__ __forceinline__ Seq seq_of(const AttendParams& p, int b) {
  Seq s;
  const int len = p.lens[b];
  s.back = false;
  s.len = min(max(len, 0), p.max_len);
  s.bad = s.len != len;
  if (p.starts) {
    const int a = p.starts[b], e = p.starts[b + 1];
    s.t0 = min(max(a, 0), p.tokens);
    const int t1 = min(max(e, s.t0), p.tokens);
    s.n = t1 - s.t0;
    s.bad = s.bad || a != s.t0 || e != t1;
    s.back = e < a;
  } else {
    s.t0 = b * p.n;
    s.n = p.n;
  }
  return s;
}
// a sequence's work: its query row tiles, each as long as its tiles of cached tokens and kSetup
// more, about what starting and storing a row tile takes (an empty sequence only stores its rows):
// 3, 5, 7 and 9 gave 66.3, 66.3, 64.5, 63.3 us (verify, 12 sequences) and 45.4, 38.7, 38.3, 39.0 (24 short ones)
template <int M>
__device__ __forceinline__ int row_tiles(const AttendParams& p, const Seq& s) {
  return (int)(((int64_t)s.n * p.heads + M - 1) / M);
}
__device__ __forceinline__ int kv_tiles(const Seq& s) { return max(1, (s.len + kN - 1) / kN); }
__device__ __forceinline__ int setup(const Seq& s) { return s.len > 0 ? kSetup : 0; }
template <int M>
__device__ __forceinline__ int work_of(const AttendParams& p, const Seq& s) {
  return row_tiles<M>(p, s) * (kv_tiles(s) + setup(s));
}

// 16-byte pieces c of LDS row r are stored at piece c ^ swz(r) (latent parts, rows of 64 pieces) or
// c ^ swz_rope(r) (rope parts, rows of 8). The LDS has 64 banks, 16 pieces. A 16-byte read serves
// lanes 0 .. 3, 12 .. 15, 20 .. 27 at once (and so on), which for the keys are 16 rows at pieces c and
// c ^ 1; a transposing read serves 32 lanes, rows r .. r + 3 and r + 8 .. r + 11 by 32 bytes. With
// these bits both meet every bank once (measured: without conflicts; with r % 16 in order, or other
// bits, one of them has some)
__device__ __forceinline__ int swz(int r) { return (r & 8) | ((r & 2) << 1) | ((r & 1) << 1); }
__device__ __forceinline__ int swz_rope(int r) { return ((r & 2) << 1) | ((r & 8) >> 2); }

// the row of tokens that are not there
__device__ const u32x4 g_zero_row[kRow * 2 / 16] = {};

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
// five of them in order, 4096 bytes apart in memory and in LDS: one wait for the base, M0's by the address's sum
// (MXFP8, whose bringing waves are the ones that hold up a tile: with a wait each, 48 sequences of 16384 140 to
// 143 us, so 133 to 135; the bf16 cache's eight rows gain nothing by it)
__device__ __forceinline__ void lds_dma16_five(const void* base, uint32_t at, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1\n\t"
      "s_add_u32 m0, m0, 0x1000\n\tv_add_u32 %0, 0x1000, %0\n\tglobal_load_lds_dwordx4 %0, %1\n\t"
      "s_add_u32 m0, m0, 0x1000\n\tv_add_u32 %0, 0x1000, %0\n\tglobal_load_lds_dwordx4 %0, %1\n\t"
      "s_add_u32 m0, m0, 0x1000\n\tv_add_u32 %0, 0x1000, %0\n\tglobal_load_lds_dwordx4 %0, %1\n\t"
      "s_add_u32 m0, m0, 0x1000\n\tv_add_u32 %0, 0x1000, %0\n\tglobal_load_lds_dwordx4 %0, %1"
      : "+v"(at)
      : "s"(base), "s"(lds)
      : "memory", "m0", "scc");
}
__device__ __forceinline__ void lds_dma4(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(lds) : "memory", "m0");
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

// v, which the compiler then forms anew where it is used: lane constants that it kept in
// registers across the tile loop cost more there than the few instructions that make them
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// a value joined over the four lanes of a column (lane % 16), in each of them
template <class F>
__device__ __forceinline__ float over_groups(float v, F join) {
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  v = join(u2f(a[0]), u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return join(u2f(b[0]), u2f(b[1]));
}
// LDS at a byte offset
template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(MKMOE_LDS const T*)(uintptr_t)at;
}

template <int M, bool MX>
struct __align__(256) AttendSmem {
  uint8_t tile[MX ? 2 : kRing][kTileBytes];  // cached rows, bf16, swizzled pieces
  uint8_t raw[MX ? kMxRing : 1][MX ? kN * kMxRow : 16];
  uint16_t p[MX ? 1 : 2][kPParts<M, MX> * M * kPStride];  // softmax numerators of a tile [part][row][token]
  float mx[M * 2];             // [row][token group]: tile maxima
  float al[M];                 // the tile's rescaling of each row; at the end the maxima
  const uint8_t* addr[2][kN];  // the rows of the tile that is requested next
  int ent[kEnts][kN];          // page entries of a tile's tokens
  int start[kMaxSeqs];         // first tile of each sequence in the work
  int scan[8];
  int first[4];                // the share's first sequence: its number, t0, n, len
  int moved[4];                // a tile's flag: some row's maximum has to move
  uint8_t bad[kN];             // tokens of the tile with a non-finite latent value
};

// The absorbed attention. The work is a list of tiles: sequence by sequence, query row tile by
// row tile (M rows: consecutive (token, head) pairs), kN cached tokens each. Every workgroup
// computes the list's prefix sums itself and takes one equal contiguous share, one workgroup a CU, so
// that ragged lengths load every CU alike. A row tile inside one share is finished there; one that was
// cut leaves its running maximum, sum and fp32 outputs in the workspace for k_latent_merge.
//
// A tile: 32 rows of 576 bf16 in LDS, read once from memory for all M query rows and used twice.
// Waves 0 .. 3 score, waves 4 .. 7 bring the tiles; both share the outputs' columns so that the
// registers hold (a scoring wave has the queries there) and the MFMA has as much of either:
//   S^T = K Q^T   scoring wave (rg, tg): the rows of half rg, tokens 16 tg ..: A = K (16-byte
//                 reads of LDS; with 64 rows each serves two row blocks), B = Q^T in registers
//   P             exp2 of the scores less the rows' running maxima, [row][token] in LDS, in bf16
//                 because it is a matrix operand (kPParts); the sums stay fp32
//   O^T += V^T P^T   latent values 32 w .. of a scoring wave (32 of them), 16 of every 64 past 128 of the
//                 others (96), for every row: A = V^T by transposing LDS reads of the same tile, B = P^T
// One barrier a tile (bf16). bf16 rows go straight from memory to LDS, three tiles ahead; MXFP8 rows
// go there as they are, and waves 4 .. 7 turn the next tile's into bf16 (exact) while waves 0 .. 3 score,
// at the price of a second barrier. PAGED: pages of kN tokens or more, so that a tile lies in one, its
// page is a scalar load and its rows follow each other; without it each token's page entry is looked up,
// two tiles before its row is (pages of one token 103 us, of 64 101 us, at 48 sequences of 8192).
//
// What bounds it, by counters at 2.3 GHz (a tile's time by the difference of two lengths). bf16: memory, 32 rows
// (48 sequences of 8192, 32 heads: 101 us with the merge, 4.5 TB/s, of it about 20 us for the start, the outputs
// and the merge; a further tile 1.7 to 2.1 us, where a copy's rate gives 1.8) and 64 rows, since every row tile
// brings the sequence's rows past the L2 anew: 24 of 8192 with 128 heads read 479 MB, twice the cache, in 91 us
// (97 with the merge), 5.3 TB/s; 48 with 64 heads as many, none of them twice, in 115 (122). A further tile of 64
// rows takes 1.5 us while the cache fits the last-level cache and 1.8 beyond, 3400 to 4200 cycles, of which the
// MFMAs need 1088 a SIMD and the LDS 714 (its 192 instructions a tile 1340 at the rate that 8 waves issue them). 12 ragged sequences with 4 queries of 64 heads:
// 245 MB in 56 us (66), 4.4 TB/s. MXFP8: the codes' way through LDS (a further tile of 32 rows 1.2 us, 2700 cycles, of
// them 1059 of LDS and 544 of MFMA; 48 of 16384, 32 heads 133 to 144 us, 3.8 TB/s, of which it took 19, while
// the conversions themselves are free; 64 of up to 16384 98). Short work is bound by the chain of lengths, pages
// and queries, first tile, outputs and merge (1025 tokens: 14 us).
//
// Steps that brought it there: whole rows by ring and DMA (64 heads 380 -> 129 us), cut row tiles joined by
// many (131071 tokens 189 -> 48), latent and rope parts apart in LDS without bank conflicts and maxima that
// rarely move (verify 96 -> 73), half as many instructions a tile (MXFP8 167 -> 149), no spill beside the
// tile loop (149 -> 138), queries by way of LDS (1025 tokens 16.1 -> 13.9).
// (64 rows spill 64 to 72 bytes a lane, at a row tile's start and end, none in the loop: a reload there would wait
// for the tiles on their way.)
template <int M, bool MX, bool PAGED>
__device__ __forceinline__ void attend_share(const AttendParams& p, AttendSmem<M, MX>& sm, const Seq& own) {
  static_assert(M == 32 || M == 64, "row blocks of 16 by two token groups on 4 or 8 waves");
  constexpr int MB = M / 16;             // row blocks
  constexpr int RB = MB / 2;             // row blocks of a scoring wave
  constexpr int KS = kRow / 32;          // MFMA steps of a score: 18
  constexpr int G = 3;                   // of them whose keys are read at once
  constexpr int kPieces = kMxRow / 16;   // 16-byte pieces of an MXFP8 row: 41
  constexpr int kMxLoads = (kN * kPieces + 63) / 64;  // wave loads of an MXFP8 tile: 21
  constexpr int kLoads = MX ? (kMxLoads + 3) / 4 : 9;  // of a wave, at most
  constexpr int kRowBytes = MX ? kMxRow : 2 * kRow;
  constexpr int kAhead = MX ? kMxRing : kRing - 1;    // tiles on their way
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const bool scores = wave < 4;
  const int rg = wave & 1, tg = (wave >> 1) & 1;  // of a scoring wave
  const int lw = wave & 3;                        // of the others: their number

  // ---- the work list
  const int mine = work_of<M>(p, own);
  int inc = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(inc, d, 64);
    if (lane >= d) inc += v;
  }
  if (lane == 63) sm.scan[wave] = inc;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int v = sm.scan[i];
    if (i < wave) before += v;
    total += v;
  }
  const int share = (total + kShares - 1) / kShares;
  const int w0 = (int)min((int64_t)blockIdx.x * share, (int64_t)total), w1 = (int)min((int64_t)w0 + share, (int64_t)total);
  const int from = before + inc - mine;
  if (tid < p.seqs) {
    sm.start[tid] = from;
    if (w0 >= from && w0 < from + mine) {
      sm.first[0] = tid;
      sm.first[1] = own.t0;
      sm.first[2] = own.n;
      sm.first[3] = own.len;
    }
  }
  if (w0 >= w1) {
    if (tid == 0) p.cut[blockIdx.x].parts = 0;
    return;
  }
  __syncthreads();

  const uint32_t tiles = (uint32_t)(uintptr_t)(MKMOE_LDS uint8_t*)sm.tile[0];
  const uint32_t p_at = (uint32_t)(uintptr_t)(MKMOE_LDS uint16_t*)sm.p[0];
  const uint32_t raws = (uint32_t)(uintptr_t)(MKMOE_LDS uint8_t*)sm.raw[0];
  const uint32_t ents = (uint32_t)(uintptr_t)(MKMOE_LDS int*)sm.ent[0];
  // the lane, in the wide variant formed anew where it is used
  auto own_lane = [&]() { return M == 32 ? lane : anew(lane); };

  int b = __builtin_amdgcn_readfirstlane(sm.first[0]);
  Seq s = {__builtin_amdgcn_readfirstlane(sm.first[1]), __builtin_amdgcn_readfirstlane(sm.first[2]),
           __builtin_amdgcn_readfirstlane(sm.first[3]), false, false};
  for (int w = w0; w < w1;) {
    if (w > w0) {
      const int last = b;
      while (b + 1 < p.seqs && __builtin_amdgcn_readfirstlane(sm.start[b + 1]) <= w) ++b;
      if (b != last) s = seq_of(p, b);
    }
    const int kt = kv_tiles(s), pre = setup(s), at = w - __builtin_amdgcn_readfirstlane(sm.start[b]);
    const int rt = at / (kt + pre), unit0 = w - (at - rt * (kt + pre));  // the row tile's place in the list
    const int tile0 = max(0, w - unit0 - pre), tile1 = min(kt, w1 - unit0 - pre);
    const int r0 = rt * M, nrows = min(M, s.n * p.heads - r0);
    w = min(w1, unit0 + pre + kt);
    if (tile1 <= 0) {  // the next share begins it
      if (tid == 0 && w >= w1) p.cut[blockIdx.x].parts = 0;
      continue;
    }

    // each row's visible tokens: query token i of n sees len - n + 1 + i
    const int base = s.len - s.n + 1;
    const int lim_lo = max(0, base + over_heads(p, r0)), lim_hi = max(0, base + over_heads(p, r0 + nrows - 1));
    const int tend = min(tile1, (lim_hi + kN - 1) / kN);
    const int32_t* table = p.table + (int64_t)b * p.table_stride;
    if (lim_hi == 0) {  // nothing to see: rows of zeros, by every share that has a part of them
      for (int i = tid; i < nrows * (kL / 8); i += kThreads) {
        const int r = r0 + i / (kL / 8), qi = over_heads(p, r), h = r - qi * p.heads;
        const int64_t to = (int64_t)(s.t0 + qi) * p.o_ts + (int64_t)h * p.o_hs + 8 * (i % (kL / 8));
        store4(p, to, f32x4{0, 0, 0, 0});
        store4(p, to + 4, f32x4{0, 0, 0, 0});
        if (p.lse && i % (kL / 8) == 0) p.lse[(int64_t)(s.t0 + qi) * p.heads + h] = -kInf;
      }
      if (tid == 0 && w >= w1) p.cut[blockIdx.x].parts = 0;
      continue;
    }

    // ---- a tile's rows on their way. Its page entries come first, to the last wave (whose other
    // loads are the fewest), which turns them into the rows' addresses well before the loads
    auto entries = [&](int t) {
      if constexpr (!PAGED) {
        const int ln = anew(lane), tok = min(t * kN + ln, lim_hi - 1);
        if (wave == 7 && ln < kN) lds_dma4(table + (tok >> p.page_shift), ents + (t % kEnts) * (4 * kN));
      }
    };
    bool lost = false;  // a page outside the cache
    auto address = [&](int tok, int pg) -> const uint8_t* {
      const bool real = tok < lim_hi, in = (uint32_t)pg < (uint32_t)p.pages;
      lost = lost || (real && !in);
      const uint32_t row = ((uint32_t)pg << p.page_shift) + (tok & ((1 << p.page_shift) - 1));
      return real && in ? p.cache + (uint64_t)row * kRowBytes : (const uint8_t*)g_zero_row;
    };
    auto resolve = [&](int t) {
      if constexpr (!PAGED) {
        const int ln = anew(lane);
        if (wave == 7 && ln < kN) sm.addr[t & 1][ln] = address(t * kN + ln, sm.ent[t % kEnts][ln]);
      }
    };
    // (PAGED) the page of tile t, by a scalar load
    typedef const int32_t __attribute__((address_space(4))) scalar_int;
    scalar_int* s_table = (scalar_int*)(uintptr_t)table;
    auto page_of = [&](int t) -> int {
      return PAGED ? s_table[min(t * kN, lim_hi - 1) >> p.page_shift] : 0;
    };
    // requests tile t: PAGED by its page, else by its rows' addresses in addr. whole: all its tokens
    // are there
    auto issue = [&](int t, int pg, const uint8_t* const* addr, bool whole) {
      const bool in = !PAGED || (uint32_t)pg < (uint32_t)p.pages;
      const uint8_t* base = nullptr;
      const int left = whole ? kN : lim_hi - t * kN;
      if (PAGED) {
        lost = lost || !in;
        const uint32_t row = ((uint32_t)pg << p.page_shift) + ((t * kN) & ((1 << p.page_shift) - 1));
        base = p.cache + (uint64_t)row * kRowBytes;
      }
      if constexpr (MX) {  // load i of wave l is number 4 i + l of the tile's 1 KB pieces
        const uint32_t dst = raws + (t - tile0) % kMxRing * (kN * kMxRow) + lw * 1024;
        const int ln = own_lane();
        const bool ends = lw < kMxLoads % 4 && ln < kN * kPieces % 64;  // the last load, not a whole one
        if (PAGED && whole && in) {
          const uint32_t at = (lw * 64 + ln) << 4;
          static_assert(kLoads == 6, "five loads, and one wave's sixth");
          lds_dma16_five(base, at, dst);
          if (ends) lds_dma16(base, at + (kLoads - 1) * 4096, dst + (kLoads - 1) * 4096);
        } else {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const uint32_t at = i * 256 + lw * 64 + ln, r = min(at / kPieces, (uint32_t)kN - 1);
            const uint8_t* row = !PAGED ? addr[r] : in && (int)r < left ? base + r * kRowBytes : (const uint8_t*)g_zero_row;
            if (i < kLoads - 1 || ends) lds_dma16(row + ((at - r * kPieces) << 4), dst + i * 4096);
          }
        }
      } else {  // wave l: the rows 8 l .. 8 l + 7, a load each and one for their rope parts
        const uint32_t dst = tiles + (t - tile0) % kRing * kTileBytes, to = dst + 8 * lw * (2 * kL);
        const uint32_t rope_to = dst + kRopeAt + 8 * lw * (2 * kR);
        const int ln = own_lane(), r = 8 * lw + (ln >> 3);
        const uint32_t at = (ln ^ swz(8 * (lw & 1))) << 4, rope_at = 2 * kL + (((ln & 7) ^ swz_rope(r)) << 4);
        if (PAGED && whole && in) {
          base += 8 * lw * kRowBytes;
#pragma unroll
          for (int i = 0; i < 8; ++i) lds_dma16(base, (at ^ (swz(i) << 4)) + i * kRowBytes, to + i * (2 * kL));
          lds_dma16(base, (ln >> 3) * kRowBytes + rope_at, rope_to);
        } else {
          const uint64_t row = PAGED ? 0 : (uint64_t)addr[r];
          const uint32_t lo = (uint32_t)row, hi = (uint32_t)(row >> 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint8_t* from;
            if (PAGED)
              from = in && 8 * lw + i < left ? base + (8 * lw + i) * kRowBytes : (const uint8_t*)g_zero_row;
            else
              from = (const uint8_t*)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, 8 * i) << 32) |
                                      (uint32_t)__builtin_amdgcn_readlane(lo, 8 * i));
            lds_dma16(from, at ^ (swz(i) << 4), to + i * (2 * kL));
          }
          const uint8_t* from = !PAGED            ? (const uint8_t*)row
                                : in && r < left ? base + r * kRowBytes
                                                 : (const uint8_t*)g_zero_row;
          lds_dma16(from + rope_at, rope_to);
        }
      }
    };
    // (waves 4 .. 7) the raw rows of tile t as bf16: 16 threads a row, the codes 8 c .. of every 128 each, so
    // that the 16 lanes which a store serves at once meet every bank once
    auto unpack = [&](int t) {
      if constexpr (MX) {
        const int ln = own_lane(), c = ln & 15;
        const uint32_t raw = raws + (t - tile0) % kMxRing * (kN * kMxRow), tile = tiles + ((t - tile0) & 1) * kTileBytes;
        const int r0 = 8 * lw + (ln >> 4), rp = 8 * lw + (ln >> 3), j = ln & 7;  // the rows r0, r0 + 4; rope parts
        const uint32_t src = raw + r0 * kMxRow;
        u32x4 scales[2];
        u32x2 q[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          scales[i] = lds_read<u32x4>(src + 4 * i * kMxRow + kL);
#pragma unroll
          for (int k = 0; k < 4; ++k) q[i][k] = lds_read<u32x2>(src + 4 * i * kMxRow + 128 * k + 8 * c);
        }
        const u32x4 pe = lds_read<u32x4>(raw + rp * kMxRow + kL + kMxScales + 16 * j);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t dst = tile + r0 * (2 * kL) + ((c ^ swz(r0)) << 4);  // (swz(r0 + 4) is swz(r0))
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)  // (the scale's byte, 4 k + c / 4)
            *(MKMOE_LDS u32x4*)(uintptr_t)(dst + 4 * i * (2 * kL) + 256 * k) =
                fp8x8(q[i][k].x, q[i][k].y, e8m0(scales[i][k] >> (8 * (c >> 2)) & 0xff));
        *(MKMOE_LDS u32x4*)(uintptr_t)(tile + kRopeAt + rp * (2 * kR) + ((j ^ swz_rope(rp)) << 4)) = pe;
      }
    };
    // waits until the tile after which `newer` more were requested has landed
    auto landed = [&](int newer) {
      if (newer <= 0) {
        wait_loads<0>();
      } else if (MX && lw >= kMxLoads % 4) {
        if (newer == 1) wait_loads<kLoads - 1>();
        else wait_loads<2 * (kLoads - 1)>();
      } else {
        if (newer == 1) wait_loads<kLoads>();
        else wait_loads<2 * kLoads>();
      }
    };

    // ---- what both kinds of wave do with a tile
    auto tile_at = [&](int t) { return tiles + (MX ? (t - tile0) & 1 : (t - tile0) % kRing) * kTileBytes; };
    constexpr int kPBytes = M * kPStride * 2;  // of a part
    auto p_of = [&](int t) { return p_at + (MX ? 0 : (t & 1) * (kPParts<M, MX> * kPBytes)); };
    // tokens that only some of the rows see: their non-finite values must not reach the others
    // through 0 * V. They are cleared, and the rows that see them become NaN
    const bool edges = lim_lo < lim_hi;
    auto sanitize = [&](int t) {
      for (int i = 0; i < kN / 8; ++i) {
        const int r = wave * (kN / 8) + i;
        u32x4* at = (u32x4*)(sm.tile[0] + (tile_at(t) - tiles) + r * (2 * kL) + (lane << 4));
        u32x4 v = *at;
        bool any = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((v[k] & 0x7f80u) == 0x7f80u) any = true, v[k] &= 0xffff0000u;
          if ((v[k] & 0x7f800000u) == 0x7f800000u) any = true, v[k] &= 0x0000ffffu;
        }
        if (t * kN + r < lim_lo) any = false;
        if (any) *at = v;
        const bool some = __any(any);
        if (lane == 0) sm.bad[r] = some;
      }
      barrier();
    };
    // V^T of the blocks of 16 latent values own + k + step c (k a multiple of what own stays under):
    // rows 8 g + col / 4 (and + 4), 4 values from 4 (lane % 4) of each block
    auto values = [&](uint32_t tile, int own, auto first, auto step, auto& va) __attribute__((always_inline)) {
      constexpr int k = decltype(first)::value, by = decltype(step)::value;
      const int ln = own_lane(), vtok = 8 * (ln >> 4) + ((ln & 15) >> 2);
      const uint32_t x = ((((ln & 3) >> 1) ^ swz(vtok)) ^ (2 * own)) << 4, row = tile + vtok * (2 * kL) + 8 * (ln & 1);
      constexpr int C = sizeof(va) / sizeof(va[0]);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int n = k + by * c;
        const uint32_t at = (x ^ ((n & 7) << 5)) + row + (n >> 3) * 256;
        struct { i16x4 a, b; } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((MKMOE_LDS i16x4*)(uintptr_t)at),
                                       __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (MKMOE_LDS i16x4*)(uintptr_t)(at + 4 * (2 * kL)))};
        va[c] = __builtin_bit_cast(bf16x8, both);
      }
    };
    auto numerators_of = [&](int t, bf16x8(&pb)[kPParts<M, MX>][MB]) {
      const int ln = own_lane();
      const uint32_t at = p_of(t) + (ln & 15) * (2 * kPStride) + ((ln >> 4) << 4);
#pragma unroll
      for (int k = 0; k < kPParts<M, MX>; ++k)
#pragma unroll
        for (int i = 0; i < MB; ++i) pb[k][i] = lds_read<bf16x8>(at + k * kPBytes + i * 16 * (2 * kPStride));
    };
    auto rescale = [&](auto& o) {
      constexpr int C = sizeof(o) / sizeof(o[0]);
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const float alpha = sm.al[16 * i + col];
#pragma unroll
        for (int c = 0; c < C; ++c) o[c][i] *= alpha;
      }
    };
    auto add = [&](auto& o, auto& va, bf16x8(&pb)[kPParts<M, MX>][MB]) {
      constexpr int C = sizeof(o) / sizeof(o[0]);
#pragma unroll
      for (int k = kPParts<M, MX> - 1; k >= 0; --k)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int c = 0; c < C; ++c) o[c][i] = mfma(va[c], pb[k][i], o[c][i]);
    };
    const bool whole = tile0 == 0 && tile1 == kt;
    const int slot = 2 * blockIdx.x + (tile0 == 0 ? 1 : 0);
    float* sums = (float*)sm.p[0];  // at the end: [row][token group]
    // the rows out: latent values first + by c .. of every row
    auto store = [&](auto& o, int first, int by, bool lead) {
      constexpr int C = sizeof(o) / sizeof(o[0]);
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int ln = anew(lane), g = ln >> 4, r = 16 * i + (ln & 15);
        if (r >= nrows) continue;
        const float sum = sums[2 * r] + sums[2 * r + 1], top = sm.al[r];
        if (whole) {
          const int qi = over_heads(p, r0 + r), h = (r0 + r) - qi * p.heads;
          const bool none = base + qi <= 0;
          const float inv = none ? 0.0f : 1.0f / sum;
          const int64_t to = (int64_t)(s.t0 + qi) * p.o_ts + (int64_t)h * p.o_hs + first + 4 * g;
#pragma unroll
          for (int c = 0; c < C; ++c) store4(p, to + by * c, o[c][i] * inv);
          if (p.lse && lead && g == 0)
            p.lse[(int64_t)(s.t0 + qi) * p.heads + h] = none ? -kInf : (top + log2f(sum)) * (1.0f / kLog2e);
        } else {
          float* dst = p.part_o + ((int64_t)slot * M + r) * kL + first + 4 * g;
#pragma unroll
          for (int c = 0; c < C; ++c) *(f32x4*)(dst + by * c) = o[c][i];
          if (lead && g == 0) {
            p.part_ml[((int64_t)slot * M + r) * 2] = top;
            p.part_ml[((int64_t)slot * M + r) * 2 + 1] = sum;
          }
        }
      }
    };
    // Steady tiles: every row sees all of them, and the tiles that their requests are for exist
    const int steady_end = min(min(tend, lim_hi / kN) - kAhead - 1, lim_lo / kN);
    __syncthreads();  // the last row tile's reads of LDS are over

    if (scores) {
      // ---- the queries into registers (a row past the tile's takes the first one's: it is not stored).
      // 32 rows a tile: by way of LDS, in the place of tiles that come later, as whole rows in order.
      // Their pieces by 16 rows, straight into the registers, take 2 us, twice as long (one sequence of 1025
      // tokens 16.2 us against 14.8); 64 rows a tile gain nothing by it (verify 65 us against 73)
      constexpr bool kByLds = M == 32;
      const uint32_t place = tiles + (MX ? 0 : kRing - 1) * kTileBytes;
      if constexpr (kByLds) {
        auto row_of = [&](int j, const uint16_t* q, int64_t ts, int64_t hs) {
          const int r = 8 * wave + j, row = r0 + (r < nrows ? r : 0), i = over_heads(p, row);
          return q + (int64_t)(s.t0 + i) * ts + (int64_t)(row - i * p.heads) * hs;
        };
        const uint64_t mine = (uint64_t)row_of(lane & 7, p.ql, p.ql_ts, p.ql_hs);
        const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint8_t* row = (const uint8_t*)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32) |
                                                (uint32_t)__builtin_amdgcn_readlane(lo, j));
          lds_dma16(row, (lane ^ swz(8 * wave + j)) << 4, place + (8 * wave + j) * (2 * kL));
        }
        const int r = 8 * wave + (lane >> 3);
        lds_dma16((const uint8_t*)row_of(lane >> 3, p.qp, p.qp_ts, p.qp_hs) + (((lane & 7) ^ swz_rope(r)) << 4),
                  place + kRopeAt + 8 * wave * (2 * kR));
      }
      bf16x8 q[RB][KS];
      int lim[RB];
      float m[RB], l[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int r = (rg * RB + rb) * 16 + col;
        const int row = r0 + (r < nrows ? r : 0), i = over_heads(p, row);
        lim[rb] = r < nrows ? max(0, base + i) : 0;
        m[rb] = -kInf;
        l[rb] = 0.0f;
        if constexpr (!kByLds) {
          const uint16_t* ql = p.ql + (int64_t)(s.t0 + i) * p.ql_ts + (int64_t)(row - i * p.heads) * p.ql_hs + 8 * g;
          const uint16_t* qp = p.qp + (int64_t)(s.t0 + i) * p.qp_ts + (int64_t)(row - i * p.heads) * p.qp_hs + 8 * g;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            q[rb][ks] = *(const bf16x8*)(ks < kL / 32 ? ql + 32 * ks : qp + 32 * (ks - kL / 32));
        }
      }
      if (tid < 4) sm.moved[tid] = 0;
      f32x4 o[2][MB];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < MB; ++i) o[c][i] = f32x4{0, 0, 0, 0};
      wait_all();
      barrier();
      if constexpr (kByLds) {
        const int r = rg * 16 + col;
        const uint32_t at = place + r * (2 * kL) + ((g ^ swz(col)) << 4);
        const uint32_t pe_at = place + kRopeAt + r * (2 * kR) + ((g ^ swz_rope(col)) << 4);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          q[0][ks] = ks < kL / 32 ? lds_read<bf16x8>((at ^ ((ks & 3) << 6)) + (ks >> 2) * 256)
                                  : lds_read<bf16x8>(pe_at ^ ((ks & 1) << 6));
      }
      barrier();
      if (MX) barrier();

      auto step = [&](int t, auto is_steady) __attribute__((always_inline)) {
        constexpr bool steady = decltype(is_steady)::value;
        const int ln = own_lane(), col = ln & 15, g = ln >> 4;
        const uint32_t tile = tile_at(t);
        const bool edge = !steady && edges && (t + 1) * kN > lim_lo;
        if (edge) sanitize(t);

        // scores, and the numerators under the maximum so far
        f32x4 sc[RB];
        float top[RB], sum[RB];
        auto numerators = [&]() {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const float mu = m[rb] == -kInf ? 0.0f : m[rb];
            float e[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = __builtin_amdgcn_exp2f(sc[rb][k] - mu);
            sum[rb] = (e[0] + e[1]) + (e[2] + e[3]);
            const uint32_t to = p_of(t) + ((rg * RB + rb) * 16 + col) * (2 * kPStride) + 32 * tg + 8 * g;
            const u32x2 near = {pack_bf(e[0], e[1]), pack_bf(e[2], e[3])};
            *(MKMOE_LDS u32x2*)(uintptr_t)to = near;
            if constexpr (kPParts<M, MX> == 2)  // (infinite ones come before the maximum moves, and are not used)
              *(MKMOE_LDS u32x2*)(uintptr_t)(to + kPBytes) =
                  u32x2{pack_bf(e[0] - bf_lo(near.x), e[1] - bf_hi(near.x)), pack_bf(e[2] - bf_lo(near.y), e[3] - bf_hi(near.y))};
          }
        };
        // keys: this lane's row of the wave's 16, pieces 4 ks + g; read a few steps ahead, and no
        // further: the registers are the queries'. Two chains of sums, so that the MFMA need not wait
        f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        const uint32_t k_at = tile + (16 * tg + col) * (2 * kL) + ((g ^ swz(col)) << 4);
        const uint32_t r_at = tile + kRopeAt + (16 * tg + col) * (2 * kR) + ((g ^ swz_rope(col)) << 4);
        bf16x8 a[2][G];
        auto keys = [&](int ks0, bf16x8(&to)[G]) {
#pragma unroll
          for (int i = 0; i < G; ++i) {
            const int ks = ks0 + i;
            to[i] = ks < kL / 32 ? lds_read<bf16x8>((k_at ^ ((ks & 3) << 6)) + (ks >> 2) * 256)
                                 : lds_read<bf16x8>(r_at ^ ((ks & 1) << 6));
          }
        };
        keys(0, a[0]);
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += G) {
          if (k0 + G < KS) keys(k0 + G, a[(k0 / G + 1) % 2]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              f32x4& to = acc[RB == 2 ? rb : (k0 + i) & 1];
              to = mfma(a[(k0 / G) & 1][i], q[rb][k0 + i], to);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (RB == 1) acc[0] += acc[1];
        bf16x8 va[2], pb[kPParts<M, MX>][MB];
        values(tile, 2 * wave, std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{}, va);
        bool move = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          sc[rb] = acc[rb] * p.scale2;
          if (!steady && (t + 1) * kN > lim_lo) {  // (rows past the tile's see every token before)
            const int r = 16 * tg + 4 * g;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (edge && sm.bad[r + k]) sc[rb][k] = __builtin_nanf("");
              if (t * kN + r + k >= lim[rb]) sc[rb][k] = -kInf;
            }
          }
          top[rb] = fmaxf(fmaxf(sc[rb][0], sc[rb][1]), fmaxf(sc[rb][2], sc[rb][3]));
          move = move || top[rb] > m[rb] + kSlack;
        }
        numerators();
        if (__any(move) && ln == 0) sm.moved[t & 3] = 1;
        if (tid == 0) sm.moved[(t + 1) & 3] = 0;  // (last read before the last barrier)
        barrier();

        numerators_of(t, pb);
        if (__builtin_amdgcn_readfirstlane(sm.moved[t & 3])) {  // maxima move: the numerators again
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            top[rb] = over_groups(top[rb], [](float a, float b) { return fmaxf(a, b); });
            if (g == 0) sm.mx[((rg * RB + rb) * 16 + col) * 2 + tg] = top[rb];
          }
          barrier();
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const int r = (rg * RB + rb) * 16 + col;
            const float both = fmaxf(sm.mx[2 * r], sm.mx[2 * r + 1]);
            float al = 1.0f;
            if (both > m[rb] + kSlack) {
              al = __builtin_amdgcn_exp2f(m[rb] - both);
              m[rb] = both;
            }
            l[rb] *= al;
            if (tg == 0 && g == 0) sm.al[r] = al;
          }
          numerators();
          barrier();
          rescale(o);
          numerators_of(t, pb);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) l[rb] += sum[rb];
        add(o, va, pb);
        if (MX) barrier();
      };
      int t = tile0;
      for (; t < steady_end; ++t) step(t, std::true_type{});
      for (; t < tend; ++t) step(t, std::false_type{});

      // ---- the row sums, then the rows out
      __syncthreads();
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int r = (rg * RB + rb) * 16 + col;
        const float v = over_groups(l[rb], [](float a, float b) { return a + b; });
        if (g == 0) sums[2 * r + tg] = v;
        if (g == 0 && tg == 0) sm.al[r] = m[rb];
      }
      __syncthreads();
      if (tid == 0 && w >= w1) {
        Cut c = {0, 0, s.t0, r0, nrows, base, M, 0};
        if (tile1 < kt) {
          c.share = (unit0 + pre) / share;
          c.parts = (unit0 + pre + kt - 1) / share - c.share + 1;
        }
        p.cut[blockIdx.x] = c;
      }
      store(o, 32 * wave, 16, wave == 0);
    } else {
      // ---- the first tiles' rows
      const uint8_t** first = (const uint8_t**)sm.p[0];  // [kAhead][kN] (P is not in use yet)
      static_assert(M * kPStride * 2 >= kAhead * kN * 8, "the first tiles' addresses fit into P");
      int pg[kAhead + 1];
      if constexpr (PAGED) {
#pragma unroll
        for (int i = 0; i <= kAhead; ++i) pg[i] = page_of(tile0 + i);
      } else {
        const int i = tid - 256;
        if (i < (kAhead + 3) * kN) {
          const int e = table[min(tile0 * kN + i, lim_hi - 1) >> p.page_shift];
          if (i < kAhead * kN) first[i] = address(tile0 * kN + i, e);
          else sm.ent[(tile0 + i / kN) % kEnts][i % kN] = e;
        }
        wait_all();
        barrier();
      }
      // (PAGED: the first tile, and the others behind the queries)
      if (PAGED) {
        issue(tile0, pg[0], first, false);
        barrier();
      }
#pragma unroll
      for (int i = PAGED; i < kAhead; ++i)
        if (tile0 + i < tend) issue(tile0 + i, pg[i], first + i * kN, false);
      int pg_next = pg[kAhead];  // the page of the tile that is requested next
      if (tile0 + kAhead < tend) resolve(tile0 + kAhead);
      if (MX && tile0 + kAhead + 1 < tend) resolve(tile0 + kAhead + 1);
      f32x4 o[6][MB];
#pragma unroll
      for (int c = 0; c < 6; ++c)
#pragma unroll
        for (int i = 0; i < MB; ++i) o[c][i] = f32x4{0, 0, 0, 0};
      landed(min(tend - 1 - tile0, kAhead - 1) - (MX ? 1 : 0));  // the first tile (MXFP8: two)
      barrier();
      if constexpr (MX) {
        if (tile0 < tend) unpack(tile0);
        barrier();
        if (tile0 + kAhead < tend) {
          entries(tile0 + kAhead + 3);
          issue(tile0 + kAhead, pg_next, sm.addr[(tile0 + kAhead) & 1], false);
          pg_next = page_of(tile0 + kAhead + 1);
        }
      }

      auto step = [&](int t, auto is_steady) __attribute__((always_inline)) {
        constexpr bool steady = decltype(is_steady)::value;
        if (!steady && edges && (t + 1) * kN > lim_lo) sanitize(t);
        bf16x8 va[6], pb[kPParts<M, MX>][MB];
        // MXFP8: the next tile takes the place of t - 1
        if (MX && (steady || t + 1 < tend)) unpack(t + 1);
        values(tile_at(t), lw, std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{}, va);
        // tile t + 1 is there at the barrier, and the one that takes the place of t - 1 (MXFP8: of the raw
        // t + 1) is requested after it
        if (!MX) landed(steady ? kAhead - 2 : min(kAhead - 2, tend - 2 - t));
        barrier();

        numerators_of(t, pb);
        if (__builtin_amdgcn_readfirstlane(sm.moved[t & 3])) {
          barrier();
          barrier();
          rescale(o);
          numerators_of(t, pb);
        }
        if (steady || t + kAhead + (MX ? 2 : 1) < tend) resolve(t + kAhead + (MX ? 2 : 1));
        constexpr int kNext = kAhead + (MX ? 1 : 0);
        if (steady || t + kNext < tend) {
          entries(t + kNext + 3);
          issue(t + kNext, pg_next, sm.addr[(t + kNext) & 1], steady);
          pg_next = page_of(t + kNext + 1);
        }
        add(o, va, pb);
        if constexpr (MX) {  // the raw rows of t + 2 are there at the barrier
          landed(steady ? kAhead - 1 : min(kAhead - 1, tend - 3 - t));
          barrier();
        }
      };
      int t = tile0;
      for (; t < steady_end; ++t) step(t, std::true_type{});
      for (; t < tend; ++t) step(t, std::false_type{});
      if (lost) record(p.err, MKMOE_LATENT_ERR_PAGE, b);
      __syncthreads();
      __syncthreads();
      store(o, 128 + 16 * lw, 64, false);
    }
  }
}

// One share of the work, in row tiles of 32 or 64. WIDE: sequences bring more than 32 query rows on
// average; 64 rows a tile read the cache half as often (48 sequences of 8192, 64 heads: 119 us against
// 160), but start, store and join twice the rows in each share, so that less than kNarrow tiles are
// taken as 32 rows (8 sequences of 1250 26 us against 33; at 4096 tiles both take 51 to 57)
template <bool MX, bool PAGED, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void k_latent_attend(AttendParams p) {
  __shared__ AttendSmem<WIDE ? 64 : 32, MX> sm;
  const int tid = threadIdx.x;
  Seq own = {0, 0, 0, false, false};
  if (tid < p.seqs) {
    own = seq_of(p, tid);
    if (own.bad && blockIdx.x == 0) record(p.err, MKMOE_LATENT_ERR_LENGTH, tid);
  }
  // query starts that run backwards give rows to several sequences, and more work than was checked
  auto over_waves = [&](int v) {  // the sum of the waves' values
    if ((tid & 63) == 0) sm.scan[tid >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) v += sm.scan[i];
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(v);
  };
  if (p.starts) {
    const bool back = over_waves(__any(own.back));
    if (blockIdx.x == 0 && tid == 0) p.covered[0] = back ? 0 : own.t0;
    if (blockIdx.x == 0 && tid == p.seqs - 1) p.covered[1] = back ? 0 : own.t0 + own.n;
    if (back) {
      if (tid == 0) p.cut[blockIdx.x].parts = 0;
      return;
    }
  }
  if constexpr (WIDE) {
    int total = work_of<64>(p, own);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d, 64);
    total = over_waves(total);
    if (total > kNarrow) return attend_share<64, MX, PAGED>(p, sm, own);
  }
  static_assert(sizeof(AttendSmem<32, MX>) <= sizeof(AttendSmem<64, MX>), "one allocation for both");
  attend_share<32, MX, PAGED>(p, reinterpret_cast<AttendSmem<32, MX>&>(sm), own);
}

// ---------------------------------------------------------------- merge
// Row tiles that were cut, their parts joined in order at their common maximum (so that the same call
// gives the same bits). Bound by latency: the parts are 17 MB at 32 rows a tile, 33 MB at 64, and take
// 4 to 10 us with the launch. kMergeWgs workgroups at each of a tile's cuts share its items, so that a
// long sequence's many parts are read by many, and every part's load is on its way before the first is
// used: up to kFewParts, an item is a row's 128 latent values, 32 lanes; up to kMoreParts, 64 values, a
// wave, whose 4 groups of 16 lanes take every fourth part; beyond, 64 values, a workgroup, 16 groups.
// (A step of 8 sequences in 20 parts each 24.9 us so, 28.9 with 8 parts at a time by 32 lanes; 256 parts
// 8.5 us by workgroups, 12.3 by 8 groups of 32 lanes; 16 to 32 parts by workgroups 5 us more than by lanes.)
constexpr int kMergeWgs = 8;
constexpr int kFewParts = 8;
constexpr int kMoreParts = 32;

__global__ __launch_bounds__(256) void k_latent_merge(AttendParams p) {
  __shared__ float s_w[kShares], s_red[4];
  __shared__ f32x4 s_acc[16][16];
  const Cut c = p.cut[blockIdx.x];
  if (c.parts == 0) return;
  const int tid = threadIdx.x;
  const int helper = (blockIdx.x - c.share) * kMergeWgs + blockIdx.y, helpers = (c.parts - 1) * kMergeWgs;
  auto at = [&](int i, int r) { return (int64_t)(2 * (c.share + i) + (i == 0 ? 1 : 0)) * c.m + r; };
  auto store = [&](int r, int first, f32x4 acc, float top, float sum) {  // 4 values of row r
    const int qi = over_heads(p, c.r0 + r), h = (c.r0 + r) - qi * p.heads;
    const bool none = c.base + qi <= 0;
    acc *= none ? 0.0f : 1.0f / sum;
    store4(p, (int64_t)(c.t0 + qi) * p.o_ts + (int64_t)h * p.o_hs + first, acc);
    if (p.lse && first == 0) p.lse[(int64_t)(c.t0 + qi) * p.heads + h] = none ? -kInf : (top + log2f(sum)) * (1.0f / kLog2e);
  };
  if (c.parts <= kFewParts) {
    const int lane = tid & 31, grp = tid >> 5;
    for (int item = helper * 8 + grp; item < 4 * c.nrows; item += helpers * 8) {
      const int r = item >> 2, first = 128 * (item & 3) + 4 * lane;
      float mi = -kInf, li = 0.0f;
      if (lane < c.parts) {
        mi = p.part_ml[at(lane, r) * 2];
        li = p.part_ml[at(lane, r) * 2 + 1];
      }
      const float* src = p.part_o + first;
      f32x4 v[kFewParts];
#pragma unroll
      for (int i = 0; i < kFewParts; ++i)
        if (i < c.parts) v[i] = *(const f32x4*)(src + at(i, r) * kL);
      float top = mi;
#pragma unroll
      for (int d = kFewParts / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 32));
      const float w = __builtin_amdgcn_exp2f(mi - (top == -kInf ? 0.0f : top));
      float sum = w * li;
#pragma unroll
      for (int d = kFewParts / 2; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 32);
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kFewParts; ++i)
        if (i < c.parts) acc += __shfl(w, i, 32) * v[i];
      top = __shfl(top, 0, 32);
      sum = __shfl(sum, 0, 32);
      store(r, first, acc, top, sum);
    }
    return;
  }
  if (c.parts <= kMoreParts) {
    constexpr int kEach = kMoreParts / 4;
    const int lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    for (int item = helper * 4 + wave; item < 8 * c.nrows; item += helpers * 4) {
      const int r = item >> 3, first = 64 * (item & 7) + 4 * (lane & 15);
      float mi = -kInf, li = 0.0f;
      if (lane < c.parts) {
        mi = p.part_ml[at(lane, r) * 2];
        li = p.part_ml[at(lane, r) * 2 + 1];
      }
      const float* src = p.part_o + first;
      f32x4 v[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (4 * i < c.parts) v[i] = *(const f32x4*)(src + at(min(4 * i + g, c.parts - 1), r) * kL);
      float top = mi;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
      const float w = __builtin_amdgcn_exp2f(mi - (top == -kInf ? 0.0f : top));
      float sum = w * li;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (4 * i < c.parts) {
          const float wi = __shfl(w, 4 * i + g, 64);
          if (4 * i + g < c.parts) acc += wi * v[i];
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = over_groups(acc[k], [](float a, float b) { return a + b; });
      if (g == 0) store(r, first, acc, top, sum);
    }
    return;
  }
  const int lane = tid & 15, grp = tid >> 4;
  for (int item = helper; item < 8 * c.nrows; item += helpers) {
    const int r = item >> 3, first = 64 * (item & 7) + 4 * lane;
    float mi = -kInf, li = 0.0f;
    if (tid < c.parts) {
      mi = p.part_ml[at(tid, r) * 2];
      li = p.part_ml[at(tid, r) * 2 + 1];
    }
    float top = mi;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((tid & 63) == 0) s_red[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, s_red[i]);
    const float w = __builtin_amdgcn_exp2f(mi - (top == -kInf ? 0.0f : top));
    s_w[tid] = w;
    float sum = w * li;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
    __syncthreads();
    if ((tid & 63) == 0) s_red[tid >> 6] = sum;
    const float* src = p.part_o + first;
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll 8
    for (int i = grp; i < c.parts; i += 16) acc += s_w[i] * *(const f32x4*)(src + at(i, r) * kL);
    s_acc[grp][lane] = acc;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int i = 1; i < 16; ++i) acc += s_acc[i][lane];
      store(r, first, acc, top, (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]));
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- the heads' products
struct ProjectParams {
  const void* x;      // bf16; fp32 (f32) where the attended latents come unrounded
  const uint16_t* w;  // [heads][256][512]: rows 0 .. 127 W_UK, 128 .. 255 W_UV
  uint16_t* y;
  int64_t x_ts, x_hs, y_ts, y_hs;
  int tokens, heads, f32;
  const int32_t* covered;  // expand in a step with query starts: the rows that attend wrote, NULL: all.
                           // The others' x is an earlier call's, and their y stays as it was
};

// what bf16's rounding left of a value, nothing where that is not finite
__device__ __forceinline__ float rest(float x, float rounded) { return fabsf(rounded) < kInf ? x - rounded : 0.0f; }

// In both products a head's workgroups are the number of heads apart, so that with 8 or a multiple of
// 8 heads they share an XCD's L2, where the head's rows are then read once: 8 XCDs that each read every
// row took 11 us for 48 tokens of 64 heads

// y[t, h, l] = sum_d x[t, h, d] W_UK[h, d, l]: a workgroup a head, 64 columns and 64 tokens; the
// 128 x 64 weight block in LDS, its transposing reads the A operand, 16 tokens a wave. The result
// is rounded to bf16 because it is the scores' matrix operand
constexpr int kAbsorbStride = 144;  // bytes an LDS row of 64 values: 16 past the banks' period
__device__ __forceinline__ void absorb_block(const ProjectParams& p, int block, uint8_t* wl) {
  constexpr int S = kAbsorbStride;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
  const int h = block % p.heads, c0 = block / p.heads % (kL / 64) * 64;
  const int t = block / p.heads / (kL / 64) * 64 + 16 * wave + col;
  const uint16_t* w = p.w + (int64_t)h * (kNope + kV) * kL + c0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = i * 256 + tid, d = at >> 3, c = at & 7;
    *(u32x4*)(wl + d * S + 16 * c) = *(const u32x4*)(w + (int64_t)d * kL + 8 * c);
  }
  const bool real = t < p.tokens;
  const uint16_t* x = (const uint16_t*)p.x + (int64_t)(real ? t : 0) * p.x_ts + (int64_t)h * p.x_hs + 8 * g;
  bf16x8 xb[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) xb[ks] = real ? *(const bf16x8*)(x + 32 * ks) : bf16x8{};
  __syncthreads();
  if (t - col >= p.tokens) return;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const uint8_t* at = wl + (32 * ks + 8 * g + (col >> 2)) * S + 32 * c + 8 * (lane & 3);
      struct { i16x4 a, b; } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((MKMOE_LDS i16x4*)at),
                                     __builtin_amdgcn_ds_read_tr16_b64_v4i16((MKMOE_LDS i16x4*)(at + 4 * S))};
      acc = mfma(__builtin_bit_cast(bf16x8, both), xb[ks], acc);
    }
    if (real)
      *(u32x2*)(p.y + (int64_t)t * p.y_ts + (int64_t)h * p.y_hs + c0 + 16 * c + 4 * g) =
          u32x2{pack_bf(acc[0], acc[1]), pack_bf(acc[2], acc[3])};
  }
}

__global__ __launch_bounds__(256) void k_latent_absorb(ProjectParams p) {
  __shared__ __align__(16) uint8_t wl[kNope * kAbsorbStride];
  absorb_block(p, blockIdx.x, wl);
}

// A step's first launch: the two that need nothing of each other, append and absorb
template <bool MX>
__global__ __launch_bounds__(256) void k_latent_front(AppendParams a, ProjectParams p, int absorb_blocks) {
  __shared__ __align__(16) uint8_t wl[kNope * kAbsorbStride];
  if ((int)blockIdx.x < absorb_blocks)
    absorb_block(p, blockIdx.x, wl);
  else
    append_block<MX, true>(a, blockIdx.x - absorb_blocks);
}

// y[t, h, j] = sum_l x[t, h, l] W_UV[h, j, l]: a workgroup a head, 16 NJ columns and 64 tokens. The
// four waves split l, so that few tokens keep them all busy and no weight is read twice, and add up
// in LDS; both operands are contiguous along l and come straight from memory. x in fp32 is taken as
// the sum of two bf16 parts (2^-17 of it is left out) against the same weights. 48 tokens of 64 heads: 7.5 us
// with 32 columns a workgroup, 9.7 with 16; 8 tokens of 32 heads 4.0 with 16
template <bool F32, int NJ>
__global__ __launch_bounds__(256) void k_latent_expand(ProjectParams p) {
  constexpr int KS = kL / 32 / 4;  // MFMA steps of a wave
  __shared__ f32x4 sums[4][NJ][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int j0 = blockIdx.y * (16 * NJ), h = blockIdx.x, t0 = blockIdx.z * 64, l0 = wave * (kL / 4) + 8 * g;
  const int from = p.covered ? p.covered[0] : 0, upto = p.covered ? min(p.covered[1], p.tokens) : p.tokens;
  const uint16_t* w = p.w + ((int64_t)h * (kNope + kV) + kNope + j0 + col) * kL + l0;
  // every operand on its way before the first is used
  using X = std::conditional_t<F32, f32x4, u32x4>;
  constexpr int kX = F32 ? 2 : 1;
  bf16x8 a[NJ][KS];
  X x[4][KS][kX];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) a[j][ks] = *(const bf16x8*)(w + 16 * j * kL + 32 * ks);
#pragma unroll
  for (int tb = 0; tb < 4; ++tb) {
    if (tb > 0 && t0 + 16 * tb >= p.tokens) continue;
    const int t = min(t0 + 16 * tb + col, p.tokens - 1);
    const int64_t at = (int64_t)t * p.x_ts + (int64_t)h * p.x_hs + l0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < kX; ++i)
        x[tb][ks][i] = *(const X*)((const uint8_t*)p.x + (at + 32 * ks) * (F32 ? 4 : 2) + 16 * i);
  }
#pragma unroll
  for (int tb = 0; tb < 4; ++tb) {
    if (tb > 0 && t0 + 16 * tb >= p.tokens) continue;
    f32x4 acc[NJ] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (F32) {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a0 = x[tb][ks][i >> 1][2 * (i & 1)], a1 = x[tb][ks][i >> 1][2 * (i & 1) + 1];
          hi[i] = pack_bf(a0, a1);
          lo[i] = pack_bf(rest(a0, bf_lo(hi[i])), rest(a1, bf_hi(hi[i])));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          acc[j] = mfma(a[j][ks], __builtin_bit_cast(bf16x8, lo), acc[j]);
          acc[j] = mfma(a[j][ks], __builtin_bit_cast(bf16x8, hi), acc[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = mfma(a[j][ks], __builtin_bit_cast(bf16x8, x[tb][ks][0]), acc[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) sums[tb][j][wave][lane] = acc[j];
  }
  __syncthreads();
  const int t = t0 + 16 * wave + col;
  if (t < from || t >= upto) return;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const f32x4* part = &sums[wave][j][0][lane];
    const f32x4 v = (part[0] + part[64]) + (part[128] + part[192]);
    *(u32x2*)(p.y + (int64_t)t * p.y_ts + (int64_t)h * p.y_hs + j0 + 16 * j + 4 * g) =
        u32x2{pack_bf(v[0], v[1]), pack_bf(v[2], v[3])};
  }
}

// ---------------------------------------------------------------- host
constexpr size_t kCtlBytes = 256, kCoveredAt = 64;  // the error words, the covered rows
constexpr size_t kCutBytes = kShares * sizeof(Cut);
constexpr size_t kMlBytes = (size_t)2 * kShares * kRowsMax * 2 * 4;
constexpr size_t kPartBytes = (size_t)2 * kShares * kRowsMax * kL * 4;
constexpr size_t kWsBytes = kCtlBytes + kCutBytes + kMlBytes + kPartBytes;
constexpr int64_t kMaxRows = (int64_t)1 << 24;  // query rows (tokens x heads) and tokens a call

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

inline int check_ws(const void* ws, size_t bytes) {
  if (!ws) return MKMOE_ERR_NULL;
  if (!aligned(ws, 256)) return MKMOE_ERR_ALIGN;
  return bytes < kWsBytes ? MKMOE_ERR_WORKSPACE : MKMOE_OK;
}
inline int check_cache(const mkmoe_latent_cache& c) {
  if (!c.data) return MKMOE_ERR_NULL;
  if (!aligned(c.data, 16)) return MKMOE_ERR_ALIGN;
  if (c.fmt != MKMOE_LATENT_BF16 && c.fmt != MKMOE_LATENT_MXFP8) return MKMOE_ERR_ARG;
  if (c.page_size < 1 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)) != 0) return MKMOE_ERR_ARG;
  if (c.pages < 1 || c.pages > (int64_t)0x7fffffff / c.page_size) return MKMOE_ERR_ARG;
  return MKMOE_OK;
}
inline int launched() { return hipGetLastError() == hipSuccess ? MKMOE_OK : MKMOE_ERR_LAUNCH; }

template <bool MX, bool PAGED>
void attend(const AttendParams& p, bool wide, hipStream_t st) {
  if (wide)
    hipLaunchKernelGGL((k_latent_attend<MX, PAGED, true>), dim3(kShares), dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((k_latent_attend<MX, PAGED, false>), dim3(kShares), dim3(kThreads), 0, st, p);
}

// the checks of each call and, where they pass, its kernel's parameters
inline int append_params(const mkmoe_latent_append_io* io, void* ws, size_t ws_bytes, AppendParams& p) {
  if (!io) return MKMOE_ERR_NULL;
  if (int rc = check_ws(ws, ws_bytes)) return rc;
  if (int rc = check_cache(io->cache)) return rc;
  if (!io->kv || !io->cos_sin || !io->positions || !io->slots) return MKMOE_ERR_NULL;
  if (io->tokens < 0 || io->tokens > kMaxRows) return MKMOE_ERR_ROWS;
  if (io->heads < 0 || io->heads > MKMOE_LATENT_MAX_HEADS || (io->rope & ~1) != 0 ||
      (io->q_out_nan & ~1) != 0 || (io->index_bytes != 4 && io->index_bytes != 8) || io->cos_sin_rows < 1 || !(io->norm_eps >= 0.0f) ||
      !isfinite(io->norm_eps) || io->kv_stride < kRow)
    return MKMOE_ERR_ARG;
  if (io->heads > 0 && (!io->q_pe || !io->q_out)) return MKMOE_ERR_NULL;
  if (!aligned(io->kv, 16) || !aligned(io->norm_w, 16) || !aligned(io->cos_sin, 16) || io->kv_stride % 8 ||
      !aligned(io->positions, io->index_bytes) || !aligned(io->slots, io->index_bytes))
    return MKMOE_ERR_ALIGN;
  if (io->heads > 0 && (!aligned(io->q_pe, 16) || !aligned(io->q_out, 16) ||
                        !strides8(io->q_token_stride, io->q_head_stride) ||
                        !strides8(io->out_token_stride, io->out_head_stride)))
    return MKMOE_ERR_ALIGN;
  if (io->heads > 0 && !rows_apart(io->out_token_stride, io->tokens, io->out_head_stride, io->heads, kR))
    return MKMOE_ERR_ARG;
  p.kv = (const uint16_t*)io->kv;
  p.norm_w = (const uint16_t*)io->norm_w;
  p.cos_sin = (const float*)io->cos_sin;
  p.positions = io->positions;
  p.slots = io->slots;
  p.q = (const uint16_t*)io->q_pe;
  p.q_out = (uint16_t*)io->q_out;
  p.cache = (uint8_t*)io->cache.data;
  p.err = (int32_t*)ws;
  p.kv_stride = io->kv_stride;
  p.q_ts = io->q_token_stride;
  p.q_hs = io->q_head_stride;
  p.o_ts = io->out_token_stride;
  p.o_hs = io->out_head_stride;
  p.rows = io->cache.pages * io->cache.page_size;
  p.table_rows = io->cos_sin_rows;
  p.tokens = io->tokens;
  p.heads = io->heads;
  p.half = io->rope == MKMOE_ROPE_HALF;
  p.wide = io->index_bytes == 8;
  p.kv_blocks = (io->tokens + 3) / 4;
  p.mark = io->q_out_nan;
  p.eps = io->norm_eps;
  return MKMOE_OK;
}
inline unsigned append_blocks(const AppendParams& p) {
  return (unsigned)(p.kv_blocks + ((int64_t)p.tokens * p.heads + 31) / 32);
}
inline int attend_params(const mkmoe_latent_attend_io* io, void* ws, size_t ws_bytes, AttendParams& p) {
  if (!io) return MKMOE_ERR_NULL;
  if (int rc = check_ws(ws, ws_bytes)) return rc;
  if (int rc = check_cache(io->cache)) return rc;
  if (!io->q_lat || !io->q_pe || !io->table || !io->lens || !io->out) return MKMOE_ERR_NULL;
  if (io->seqs < 1 || io->seqs > kMaxSeqs || io->tokens < 0) return MKMOE_ERR_ROWS;
  if (io->heads < 1 || io->heads > MKMOE_LATENT_MAX_HEADS) return MKMOE_ERR_ARG;
  if ((int64_t)io->tokens * io->heads > kMaxRows) return MKMOE_ERR_ROWS;
  if (!io->q_starts && io->tokens % io->seqs != 0) return MKMOE_ERR_ROWS;
  if ((io->out_f32 & ~1) != 0) return MKMOE_ERR_ARG;
  if (!isfinite(io->scale) || io->max_pages < 1 || io->table_stride < io->max_pages) return MKMOE_ERR_ARG;
  const int64_t max_len = (int64_t)io->max_pages * io->cache.page_size;
  if (max_len > (int64_t)1 << 30) return MKMOE_ERR_ARG;
  // the work list's tiles are counted in 32 bits
  const int64_t tiles = ((int64_t)io->tokens * io->heads / 32 + io->seqs) * ((max_len + kN - 1) / kN + kSetup);
  if (tiles > 0x3fffffff) return MKMOE_ERR_ARG;
  const void* wide[] = {io->q_lat, io->q_pe, io->out};
  for (const void* q : wide)
    if (!aligned(q, 16)) return MKMOE_ERR_ALIGN;
  const void* narrow[] = {io->table, io->lens, io->q_starts, io->lse};
  for (const void* q : narrow)
    if (!aligned(q, 4)) return MKMOE_ERR_ALIGN;
  if (!strides8(io->ql_token_stride, io->ql_head_stride) || !strides8(io->qp_token_stride, io->qp_head_stride) ||
      !strides8(io->out_token_stride, io->out_head_stride))
    return MKMOE_ERR_ALIGN;
  if (!rows_apart(io->out_token_stride, io->tokens, io->out_head_stride, io->heads, kL)) return MKMOE_ERR_ARG;
  p.ql = (const uint16_t*)io->q_lat;
  p.qp = (const uint16_t*)io->q_pe;
  p.cache = (const uint8_t*)io->cache.data;
  p.table = io->table;
  p.lens = io->lens;
  p.starts = io->q_starts;
  p.out = io->out;
  p.f32 = io->out_f32;
  p.lse = io->lse;
  uint8_t* at = (uint8_t*)ws;
  p.err = (int32_t*)at;
  p.covered = (int32_t*)(at + kCoveredAt);
  p.cut = (Cut*)(at += kCtlBytes);
  p.part_ml = (float*)(at += kCutBytes);
  p.part_o = (float*)(at += kMlBytes);
  p.ql_ts = io->ql_token_stride;
  p.ql_hs = io->ql_head_stride;
  p.qp_ts = io->qp_token_stride;
  p.qp_hs = io->qp_head_stride;
  p.o_ts = io->out_token_stride;
  p.o_hs = io->out_head_stride;
  p.table_stride = io->table_stride;
  p.pages = (int)io->cache.pages;
  p.seqs = io->seqs;
  p.tokens = io->tokens;
  p.heads = io->heads;
  p.n = io->q_starts ? 0 : io->tokens / io->seqs;
  p.max_len = (int)max_len;
  p.page_shift = __builtin_ctz((unsigned)io->cache.page_size);
  p.per_head = (uint32_t)(((1ull << 32) + io->heads - 1) / io->heads);
  p.scale2 = io->scale * kLog2e;
  return MKMOE_OK;
}
inline int attend_launch(const mkmoe_latent_attend_io* io, const AttendParams& p, hipStream_t st) {
  if (io->tokens == 0) return MKMOE_OK;
  const bool mx = io->cache.fmt == MKMOE_LATENT_MXFP8, paged = io->cache.page_size >= kN;
  const bool wide = ((int64_t)io->tokens * io->heads + io->seqs - 1) / io->seqs > 32;
  if (mx)
    paged ? attend<true, true>(p, wide, st) : attend<true, false>(p, wide, st);
  else
    paged ? attend<false, true>(p, wide, st) : attend<false, false>(p, wide, st);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(k_latent_merge, dim3(kShares, kMergeWgs), dim3(256), 0, st, p);
  return launched();
}
inline int project_params(const mkmoe_latent_project_io* io, ProjectParams& p) {
  if (!io || !io->x || !io->w || !io->y) return MKMOE_ERR_NULL;
  if (io->tokens < 0 || io->tokens > (1 << 20)) return MKMOE_ERR_ROWS;
  if (io->heads < 1 || io->heads > MKMOE_LATENT_MAX_HEADS || (io->expand & ~1) != 0 || (io->x_f32 & ~1) != 0 ||
      (io->x_f32 && !io->expand))
    return MKMOE_ERR_ARG;
  if (!aligned(io->x, 16) || !aligned(io->w, 16) || !aligned(io->y, 16) ||
      !strides8(io->x_token_stride, io->x_head_stride) || !strides8(io->y_token_stride, io->y_head_stride))
    return MKMOE_ERR_ALIGN;
  if (!rows_apart(io->y_token_stride, io->tokens, io->y_head_stride, io->heads, io->expand ? kV : kL)) return MKMOE_ERR_ARG;
  p = ProjectParams{io->x, (const uint16_t*)io->w, (uint16_t*)io->y, io->x_token_stride, io->x_head_stride,
                    io->y_token_stride, io->y_head_stride, io->tokens, io->heads, io->x_f32, nullptr};
  return MKMOE_OK;
}
inline unsigned absorb_blocks(const ProjectParams& p) {
  return (unsigned)(kL / 64) * p.heads * ((p.tokens + 63) / 64);
}
inline int expand_launch(const ProjectParams& p, hipStream_t st) {
  // 32 columns a workgroup where that still gives every CU one
  const bool wide = p.heads * (kV / 32) >= kShares;
  const dim3 grid(p.heads, wide ? kV / 32 : kV / 16, (p.tokens + 63) / 64);
  if (p.f32 && wide)
    hipLaunchKernelGGL((k_latent_expand<true, 2>), grid, dim3(256), 0, st, p);
  else if (p.f32)
    hipLaunchKernelGGL((k_latent_expand<true, 1>), grid, dim3(256), 0, st, p);
  else if (wide)
    hipLaunchKernelGGL((k_latent_expand<false, 2>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((k_latent_expand<false, 1>), grid, dim3(256), 0, st, p);
  return launched();
}

}  // namespace mkmoe_latent

extern "C" {

int mkmoe_latent_workspace_bytes(size_t* bytes) {
  if (!bytes) return MKMOE_ERR_NULL;
  *bytes = mkmoe_latent::kWsBytes;
  return MKMOE_OK;
}

int mkmoe_latent_append(const mkmoe_latent_append_io* io, void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  AppendParams p;
  if (int rc = append_params(io, ws, ws_bytes, p)) return rc;
  if (p.tokens == 0) return MKMOE_OK;
  hipStream_t st = (hipStream_t)stream;
  if (io->cache.fmt == MKMOE_LATENT_MXFP8)
    hipLaunchKernelGGL(k_latent_append<true>, dim3(append_blocks(p)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(k_latent_append<false>, dim3(append_blocks(p)), dim3(256), 0, st, p);
  return launched();
}

int mkmoe_latent_rows(const mkmoe_latent_cache* cache, const void* slots, int32_t index_bytes, int32_t tokens, void* out,
                      void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  if (!cache || !slots || !out) return MKMOE_ERR_NULL;
  if (int rc = check_ws(ws, ws_bytes)) return rc;
  if (int rc = check_cache(*cache)) return rc;
  if (tokens < 0 || tokens > kMaxRows) return MKMOE_ERR_ROWS;
  if (index_bytes != 4 && index_bytes != 8) return MKMOE_ERR_ARG;
  if (!aligned(slots, index_bytes) || !aligned(out, 16)) return MKMOE_ERR_ALIGN;
  if (tokens == 0) return MKMOE_OK;
  RowsParams p{(const uint8_t*)cache->data, slots, (uint16_t*)out, (int32_t*)ws, cache->pages * cache->page_size, tokens,
               index_bytes == 8};
  const dim3 grid((tokens + 3) / 4);
  if (cache->fmt == MKMOE_LATENT_MXFP8)
    hipLaunchKernelGGL(k_latent_rows<true>, grid, dim3(256), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(k_latent_rows<false>, grid, dim3(256), 0, (hipStream_t)stream, p);
  return launched();
}

int mkmoe_latent_attend(const mkmoe_latent_attend_io* io, void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  AttendParams p;
  if (int rc = attend_params(io, ws, ws_bytes, p)) return rc;
  return attend_launch(io, p, (hipStream_t)stream);
}

int mkmoe_latent_project(const mkmoe_latent_project_io* io, void* stream) {
  using namespace mkmoe_latent;
  ProjectParams p;
  if (int rc = project_params(io, p)) return rc;
  if (io->tokens == 0) return MKMOE_OK;
  hipStream_t st = (hipStream_t)stream;
  if (io->expand) return expand_launch(p, st);
  hipLaunchKernelGGL(k_latent_absorb, dim3(absorb_blocks(p)), dim3(256), 0, st, p);
  return launched();
}

int mkmoe_latent_step(const mkmoe_latent_append_io* append, const mkmoe_latent_project_io* absorb,
                      const mkmoe_latent_attend_io* attend, const mkmoe_latent_project_io* expand, void* ws,
                      size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  AppendParams a;
  ProjectParams k, v;
  AttendParams s;
  if (int rc = append_params(append, ws, ws_bytes, a)) return rc;
  if (int rc = project_params(absorb, k)) return rc;
  if (int rc = attend_params(attend, ws, ws_bytes, s)) return rc;
  if (int rc = project_params(expand, v)) return rc;
  if (absorb->expand || !expand->expand) return MKMOE_ERR_ARG;
  if (append->tokens != attend->tokens || absorb->tokens != attend->tokens || expand->tokens != attend->tokens)
    return MKMOE_ERR_ROWS;
  // what one part writes is as large as what the next reads
  const mkmoe_latent_cache &from = append->cache, &to = attend->cache;
  if ((append->heads != 0 && append->heads != attend->heads) || absorb->heads != attend->heads ||
      expand->heads != attend->heads || expand->x_f32 != attend->out_f32 || from.data != to.data ||
      from.pages != to.pages || from.page_size != to.page_size || from.fmt != to.fmt)
    return MKMOE_ERR_ARG;
  if (s.tokens == 0) return MKMOE_OK;
  if (s.starts) v.covered = s.covered;
  hipStream_t st = (hipStream_t)stream;
  const int first = (int)absorb_blocks(k);
  if (append->cache.fmt == MKMOE_LATENT_MXFP8)
    hipLaunchKernelGGL(k_latent_front<true>, dim3(first + append_blocks(a)), dim3(256), 0, st, a, k, first);
  else
    hipLaunchKernelGGL(k_latent_front<false>, dim3(first + append_blocks(a)), dim3(256), 0, st, a, k, first);
  if (int rc = launched()) return rc;
  if (int rc = attend_launch(attend, s, st)) return rc;
  return expand_launch(v, st);
}

int mkmoe_latent_read_errors(const void* ws, int32_t* words, int32_t n, void* stream) {
  if (!ws || !words) return MKMOE_ERR_NULL;
  if (n < 1 || n > MKMOE_LATENT_ERRW_WORDS) return MKMOE_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (hipMemcpyAsync(words, ws, (size_t)n * 4, hipMemcpyDeviceToHost, st) != hipSuccess) return MKMOE_ERR_HIP;
  return hipStreamSynchronize(st) == hipSuccess ? MKMOE_OK : MKMOE_ERR_HIP;
}

}  // extern "C"
