// Latent attention of a prompt's tokens on gfx950 (MI355X): HIP kernels and the C ABI of the prompt
// section of include/mkmoe.h.
//
// A chunk of a sequence's new tokens attends over its cached rows, its own among them, with a key
// and a value for every head and token, made from the row's latent part c by the head's weights:
//   k = [W_UK c, k_pe] (128 + 64 values),  v = W_UV c (128),
//   s = scale (q_nope . W_UK c + q_pe . k_pe),  o = sum softmax(s) v,
// 640 operations a score where the absorbed form needs 2176, for 262144 a head and cached token once a
// call: the fewer from about 171 new tokens a sequence.
//
//   k_prompt_rows     the cached rows as they are multiplied, one sequence after the other; the plan
//   k_prompt_heads    every head's keys and values of them, a matrix product
//   k_prompt_attend   the attention, its work cut into equal shares over the card
//   k_prompt_merge    joins the shares of a query tile that was cut
//
// Operands are kept as the 32x32x16 matrix instruction takes them: a fragment is 1 KB, 16 bytes a
// lane, so that every load is linear, in memory and in LDS, and no bank conflicts arise. Lane l of one
// holds row l % 32 (a token, or an output value) and 8 of 16 values along the sum, those of half
// l / 32. Sums run over values in any order that both operands share, and a product leaves lane l
// with rows 8 i + 4 (l / 32) + j, i, j < 4, of column l % 32: the order kept here ("dealt": half
// h holds values 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3 of 16), so that a product's output is
// the next one's operand in place: keys and values are stored, and numerators used, without
// any exchange between lanes.
//
// Rounded to fewer bits than fp32 are the operands of the matrix instructions: keys to bf16, whose range
// queries need, numerators and values to fp16 (3 more bits), a tile's values to bf16 where fp16 would be coarser
// for one of them (k_prompt_heads). Against 64 bits, in the 2-norm, where the output's own rounding is 0.0017: 0.0019 to
// 0.0022 where rows see few keys (with all values in bf16 0.0028), 0.0017 over long ones. Sums, maxima, outputs and parts are fp32;
// the sums are of the numerators as they are multiplied, so that a row's weights add up to 1.
//
// Times below are of an MI355X, of passes among others. The floors are made with 4.91 TB/s, a copy of 2 GiB, and 1.39
// PFLOP/s, a bf16 product of 8192^3.

#include "mkmoe_latent.h"
#include "mkmoe_prompt_cut.h"

namespace mkmoe_latent {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// units of work that a share has at least (4, 6, 9: 193 tokens over 893 37.5, 36.1, 37.6 us)
constexpr int kLeastUnits = 6;
constexpr int kFrag = 1024;         // bytes of a fragment
constexpr int kPromptSeqs = MKMOE_LATENT_MAX_SEQS;
constexpr float kMoveBy = 8.0f;     // a row's maximum moves where a score passes it by more than 2^kMoveBy
constexpr float kLog2 = 0.69314718055994531f, kLog2E = 1.4426950408889634f;
// Values in fp16 are held 2^kValueLift above themselves, so that fp16 is no coarser than bf16 for any from 2^-26, where its
// spacing of 2^-24 is bf16's 2^-7 of them, up to kValueMost. Outputs are 2^kValueLift above themselves until they are stored
constexpr int kValueLift = 9;
constexpr float kValueUnit = 0x1p-9f, kValueLeast = 0x1p-17f * kValueUnit, kValueMost = 65504.0f * kValueUnit;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// two fp32 as fp16 (nearest even), a in the low half
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f16x2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, v);
}
// sums of numerators as they are multiplied: c + the two of w
__device__ __forceinline__ float add_f16(uint32_t w, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
}
// (bf16 ones are 2^kValueLift above fp16's, whose values are)
__device__ __forceinline__ float add_bf16(uint32_t w, float c) { return fmaf(bf_lo(w) + bf_hi(w), kValueUnit, c); }
// the largest, of scores say; NaN where one is (their row's output is NaN either way)
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ const uint8_t* uniform(const uint8_t* q) {
  const uint64_t v = (uint64_t)q;
  return (const uint8_t*)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)(uint32_t)v));
}

// where each sequence's rows and work are; written by k_prompt_rows, read by the launches behind it
struct Plan {
  int32_t at[kPromptSeqs];    // first row of the packed tokens; -1: they do not fit
  int32_t work[kPromptSeqs];  // first unit of the attention's work
  int32_t item[kPromptSeqs];  // first item of it: a head's query tile each
  int32_t first[kMaxShares];  // each share's first item
  int32_t rows;               // packed rows, a multiple of kKeys
  int32_t total;              // units of work
  int32_t per;                // units a share
  int32_t items;
  int32_t odd;                // some tile's values are bf16
  int32_t back;               // query starts run backwards
};

// what the end of a share cut, for the merge: a query tile that goes on in the shares behind it
struct PromptCut {
  int32_t parts;  // the shares behind it that have a part; 0: nothing was cut there
  int32_t head, t0, n;  // the sequence's first query token, its query tokens
  int32_t qt;
  int32_t unused[3];
};

struct PromptParams {
  const uint16_t* qn;
  const uint16_t* qp;
  const uint16_t* w;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;  // NULL: n query tokens a sequence
  uint16_t* out;
  float* lse;
  int32_t* err;
  Plan* plan;
  uint8_t* c;      // latent fragments [cap / 32][32][1 KB]
  uint8_t* pe;     // rope fragments [cap / 32][4][1 KB]
  uint8_t* k;      // key fragments [heads][cap / 32][8][1 KB]
  uint8_t* v;      // value fragments [heads][cap / 32][2][4][1 KB]
  int32_t* odd;    // [heads][cap / 64]: a tile's values are 0: fp16, 1: bf16, 2: bf16 and may not be finite
  PromptCut* cut;  // [shares]
  float* part_o;   // [2 shares][W][4][4][64 lanes][4]
  float* part_ml;  // [2 shares][32 W][2]
  int64_t qn_ts, qn_hs, qp_ts, qp_hs, o_ts, o_hs, table_stride;
  int64_t cap;     // packed rows that the workspace holds, a multiple of kKeys
  int pages, seqs, tokens, heads, n, max_len, page_shift;
  int waves;       // of the attention's workgroups
  float scale2;    // |scale| log2(e)
  uint32_t flip;   // 0x80008000 where scale is negative: the keys' signs are turned
};

// a sequence's query tokens and length, clamped to their bounds. Where query starts run backwards (back), it begins
// where those before it end: no row is two sequences', and there is no more work than was checked
struct PromptSeq {
  int t0, n, len;
  bool bad;  // outside its bounds
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int b, bool back) {
  PromptSeq s;
  const int len = p.lens[b];
  s.len = min(max(len, 0), p.max_len);
  s.bad = s.len != len;
  if (p.starts) {
    const int a = p.starts[b], e = p.starts[b + 1];
    s.t0 = a;
    for (int i = 0; back && i < b; ++i) s.t0 = max(s.t0, p.starts[i]);
    s.t0 = min(max(s.t0, 0), p.tokens);
    const int t1 = min(max(e, s.t0), p.tokens);
    s.n = t1 - s.t0;
    s.bad = s.bad || a != s.t0 || e != t1;
  } else {
    s.t0 = b * p.n;
    s.n = p.n;
  }
  return s;
}

// A head's query tiles in order, each of kItemSetup units and one for each turn of keys that its last
// row sees. Tile i sees past + rows (i + 1) keys (the last one past + n), past = len - n below 0 where there
// are more queries than cached tokens: 4 (i + 1) + turns(past) turns, for 4 turns are a query tile's rows.
__device__ __forceinline__ int turns_of(int past, int n, int i, int w) {
  return max(0, past + min(n, rows_of(w) * (i + 1)) + (1 << key_shift(w)) - 1) >> key_shift(w);
}
// units before query tile i, none of those before it the last
__device__ __forceinline__ int units_before(int past, int i, int w) {
  const int cp = (past + (1 << key_shift(w)) - 1) >> key_shift(w);  // (rounded up, below 0 too)
  const int first = cp < 0 ? (-cp) >> 2 : 0;                        // the first tile that sees a key
  int u = i * kItemSetup;
  if (i > first) u += 2 * (i * (i + 1) - first * (first + 1)) + (i - first) * cp;
  return u;
}
__device__ __forceinline__ int query_tiles(int n, int w) { return (n + rows_of(w) - 1) / rows_of(w); }
__device__ __forceinline__ int head_units(int past, int n, int w) {
  const int last = query_tiles(n, w) - 1;
  return units_before(past, last, w) + kItemSetup + turns_of(past, n, last, w);
}

// ---------------------------------------------------------------- rows
// the sum of v over the threads before this one of 256, and over all of them
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t* total, int64_t* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < wave) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return before + x - v;
}

// The packed rows, 32 tokens a workgroup and turn: a fragment a wave and turn, its lanes reading 16 bytes (MXFP8: 8
// codes) of 32 rows each; a row's lines are read once and hit the cache then. Rows behind a sequence's end are zeros, so
// that nothing there reaches its keys. Every workgroup forms the sequences' places itself; one more plans the attention: its
// work list's prefix sums and each share's first item, so that nothing is planned on the host and a captured graph replays
// with other lengths. Memory bounds it (65300 rows in bf16, 150 MB: 36 us, 4.2 TB/s), on few rows latency (893 rows 6 us).
template <bool MX>
__global__ __launch_bounds__(256) void k_prompt_rows(PromptParams p) {
  __shared__ int64_t sums[4];
  __shared__ int at[kPromptSeqs], unit[kPromptSeqs], item[kPromptSeqs];
  __shared__ int upto;  // the end of the last rows that fit
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, groups = gridDim.x - 1;
  const bool planner = (int)blockIdx.x == groups;
  int64_t rows = 0, work = 0, items = 0;
  if (tid == 0) upto = 0;  // (the scan's barriers come before it is used)
  int behind = 0;
  for (int b = tid; p.starts && b < p.seqs; b += 256) behind |= p.starts[b + 1] < p.starts[b];
  const bool back = __syncthreads_or(behind) != 0;
  for (int b0 = 0; b0 < p.seqs; b0 += 256) {
    const int b = b0 + tid;
    int need = 0;
    PromptSeq s{0, 0, 0, false};
    if (b < p.seqs) {
      s = prompt_seq(p, b, back);
      if (s.bad && planner) record(p.err, MKMOE_LATENT_ERR_LENGTH, b);
      if (s.n > 0) need = (s.len + kKeys - 1) & -kKeys;
    }
    int64_t all;
    const int64_t from = rows + scan256(need, &all, sums);
    rows += all;
    const bool fits = need == 0 || from + need <= p.cap;
    if (b < p.seqs) {
      at[b] = (int)(fits ? min(from, p.cap) : p.cap);  // (in order, to be searched)
      if (fits) atomicMax(&upto, (int)min(from + need, p.cap));
    }
    if (!planner) continue;
    int64_t units = 0, mine = 0;
    if (b < p.seqs && s.n > 0) {
      units = (int64_t)p.heads * (fits ? head_units(s.len - s.n, s.n, p.waves) : query_tiles(s.n, p.waves) * kItemSetup);
      mine = (int64_t)p.heads * query_tiles(s.n, p.waves);
    }
    const int64_t first = work + scan256(units, &all, sums);
    work += all;
    const int64_t first_item = items + scan256(mine, &all, sums);
    items += all;
    if (b < p.seqs) {
      unit[b] = p.plan->work[b] = (int)first;
      item[b] = p.plan->item[b] = (int)first_item;
      p.plan->at[b] = fits ? at[b] : -1;
      if (!fits) record(p.err, MKMOE_LATENT_ERR_CONTEXT, b);
    }
  }
  __syncthreads();
  const int end = upto;
  if (planner) {
    const int shares = shares_of(p.waves), per = (int)max((int64_t)kLeastUnits, (work + shares - 1) / shares);
    if (tid == 0) {
      p.plan->rows = end;
      p.plan->total = (int)work;
      p.plan->items = (int)items;
      p.plan->per = per;
      p.plan->odd = 0;
      p.plan->back = back;
    }
    for (int share = tid; share < shares; share += 256) {
      p.cut[share].parts = 0;  // (the attention's share says otherwise)
      const int64_t u = (int64_t)share * per;
      if (u >= work) continue;
      // the share's first item: the one that has its first unit
      int lo = 0, hi = p.seqs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (unit[mid] <= u) lo = mid; else hi = mid - 1;
      }
      const PromptSeq s = prompt_seq(p, lo, back);
      const int qts = query_tiles(s.n, p.waves), past = s.len - s.n;
      int x = (int)u - unit[lo], i = 0;
      if (at[lo] == p.cap && s.len > 0) {  // it does not fit: no keys
        i = x / kItemSetup;
      } else {
        const int head = x / head_units(past, s.n, p.waves);
        x -= head * head_units(past, s.n, p.waves);
        int a = 0, z = qts - 1;
        while (a < z) {
          const int mid = (a + z + 1) >> 1;
          if (units_before(past, mid, p.waves) <= x) a = mid; else z = mid - 1;
        }
        i = head * qts + a;
      }
      p.plan->first[share] = item[lo] + i;
    }
    return;
  }
  // (a fragment's row and half)
  const int r = lane & 31, half = lane >> 5;
  for (int kb = blockIdx.x; kb < end >> 5; kb += groups) {
    int lo = 0, hi = p.seqs - 1;  // the last sequence that starts at or before the block
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (at[mid] <= kb * 32) lo = mid; else hi = mid - 1;
    }
    const int b = lo, t = kb * 32 - at[b] + r;
    const int len = min(max(p.lens[b], 0), p.max_len);
    const uint8_t* src = nullptr;
    if (t < len) {
      const int page = p.table[(int64_t)b * p.table_stride + (t >> p.page_shift)];
      if ((uint32_t)page < (uint32_t)p.pages) {
        const int64_t row = ((int64_t)page << p.page_shift) + (t & ((1 << p.page_shift) - 1));
        src = p.cache + row * (MX ? kMxRow : 2 * kRow);
      } else if (wave == 0 && half == 0) {
        record(p.err, MKMOE_LATENT_ERR_PAGE, b);
      }
    }
    uint8_t* c = p.c + (int64_t)kb * 32 * kFrag + lane * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int ks = wave * 8 + i;
      u32x4 v = {0, 0, 0, 0};
      if (src) {
        if constexpr (MX) {
          const u32x2 q = *(const u32x2*)(src + 16 * ks + 8 * half);
          v = fp8x8(q.x, q.y, e8m0(src[kL + (ks >> 1)]));
        } else {
          v = *(const u32x4*)(src + 32 * ks + 16 * half);
        }
      }
      *(u32x4*)(c + ks * kFrag) = v;
    }
    u32x4 v = {0, 0, 0, 0};
    if (src) v = *(const u32x4*)(src + (MX ? kL + kMxScales : 2 * kL) + 32 * wave + 16 * half);
    *(u32x4*)(p.pe + ((int64_t)kb * 4 + wave) * kFrag + lane * 16) = u32x4{v.x ^ p.flip, v.y ^ p.flip, v.z ^ p.flip, v.w ^ p.flip};
  }
}

// ---------------------------------------------------------------- keys and values of every head
// The product of packed rows and kv_b. A workgroup, one a CU, keeps 128 of the weights' rows, a head's W_UK or W_UV, in
// LDS, and its 8 waves go through the tokens on their own, without barriers: 64 tokens a turn by the 128 rows (8 matrix
// instructions to 4 reads of LDS, half of what it can deliver, and 2 of memory), the tokens' fragments coming from memory
// four steps ahead, on into the next turn. Stages of tokens and weights through LDS with a barrier each took a quarter longer (300
// over 65300 677 -> 613 us a call, 8191 over 16383 178 -> 143 of it).
// Power bounds it: 16384 tokens of 32 heads, 137 GFLOP, take 135 to 143 us (0.96 to 1.02 PFLOP/s), the matrix units busy for 61 % of
// the cycles at 1.75 GHz; 65300 of 16 heads, 535 MB written, 246 to 306. 893 of 16 heads take 12: the weights' and tokens'
// first loads and one turn (32 rows a wave, four waves a turn, instead: 13).
constexpr int kHalfHead = 128 * kL * 2;  // bytes
constexpr int kAhead = 4;
template <bool V>
__device__ __forceinline__ void heads_blocks(const PromptParams& p, uint32_t lds, int head, int from, int upto) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int blk = from + wave;
  constexpr int64_t kBlockBytes = 64 * kL * 2;
  const uint8_t* at = p.c + blk * kBlockBytes;
  bf16x8 c[kAhead][2], w[2][4];
  if (blk < upto) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) c[u][t] = *(const bf16x8*)(at + t * kBlockBytes / 2 + u * kFrag + lane * 16);
  }
  // the weights, a row a load, so that its lines are read whole. A row's 16-byte pieces are in the order of their number
  // exclusive or the row's, so that reads of a fragment, a piece of 32 rows each, have no bank conflicts
  const uint8_t* rows = (const uint8_t*)(p.w + (int64_t)(2 * head + V) * 128 * kL);
  __syncthreads();  // (every wave is done with the weights before)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = wave * 16 + i;
    lds_dma16(rows + r * kL * 2, (lane ^ (r & 31)) * 16, lds + r * kL * 2);
  }
  wait_all();
  __syncthreads();
  if (blk >= upto) return;
  const uint32_t w_at = lds + (lane & 31) * kL * 2 + ((lane & 31) ^ (lane >> 5)) * 16;
  auto weight = [&](int j, int ks) { return lds_read<bf16x8>((w_at ^ (ks << 5)) + j * 32 * kL * 2); };
  for (;; blk += 8) {
    const bool more = blk + 8 < upto;
    const uint8_t* next = more ? at + 8 * kBlockBytes : at;
    f32x16 acc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t][j] = f32x16{};
#pragma unroll
    for (int j = 0; j < 4; ++j) w[0][j] = weight(j, 0);
#pragma unroll 1
    for (int k = 0; k < kL / 16; k += kAhead) {
      const uint8_t* ahead = k + kAhead < kL / 16 ? at + (k + kAhead) * kFrag : next;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int after = (k + u + 1) % (kL / 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[(u + 1) & 1][j] = weight(j, after);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[t][j] = V ? mfma32(c[u][t], w[u & 1][j], acc[t][j]) : mfma32(w[u & 1][j], c[u][t], acc[t][j]);
#pragma unroll
        for (int t = 0; t < 2; ++t) c[u][t] = *(const bf16x8*)(ahead + t * kBlockBytes / 2 + u * kFrag + lane * 16);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int64_t kb = (int64_t)head * (p.cap / 32) + 2 * blk;
    // Keys and values that the last-level cache does not hold until they are read leave it to others (300 over 65300, 535 MB:
    // 610 -> 589 us; ragged prompts' step, 130 MB: 193 -> 197)
    const bool stream = (int64_t)p.plan->rows * p.heads * 512 > 256 << 20;
    auto store_as = [&](auto pack, auto streamed) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const f32x16& a = acc[t][j];
            const u32x4 o = {pack(a[8 * u], a[8 * u + 1]), pack(a[8 * u + 2], a[8 * u + 3]), pack(a[8 * u + 4], a[8 * u + 5]),
                             pack(a[8 * u + 6], a[8 * u + 7])};
            u32x4* to = (u32x4*)((V ? p.v : p.k) + ((kb + t) * 8 + (V ? u * 4 + j : 2 * j + u)) * kFrag + lane * 16);
            if constexpr (streamed()) {
              asm volatile("");  // (or the two branches' stores become one)
              __builtin_nontemporal_store(o, to);
            } else {
              *to = o;
            }
          }
    };
    auto store = [&](auto pack) {
      if (stream)
        store_as(pack, [] { return true; });
      else
        store_as(pack, [] { return false; });
    };
    if constexpr (V) {
      // fp16 where it is no coarser than bf16 for any of the values that is not 0: a query may see one token alone, and
      // outputs are never mixed, so what a value loses is not measured by another one
      float top = 0.0f;
      uint32_t low = ~0u;  // of a size's bits, less one: 0, which is held exactly, comes last
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x = acc[t][j][i], y = acc[t][j][i + 1];
            top = max3(top, fabsf(x), fabsf(y));
            low = min(min(low, (f2u(x) << 1) - 1), (f2u(y) << 1) - 1);
          }
      const bool half = __ballot(!(top < kValueMost) || low < (f2u(kValueLeast) << 1) - 1) == 0;
      const bool finite = __ballot(!(top < 0x1p127f)) == 0;  // (in bf16, too)
      if (lane == 0) p.odd[(int64_t)head * (p.cap / kKeys) + blk] = half ? 0 : finite ? 1 : 2;
      if (half) {
        store([](float x, float y) {
          // (a fused product and sum is rounded to fp16 by the same instruction)
          return pack_f16(fmaf(x, 1.0f / kValueUnit, 0.0f), fmaf(y, 1.0f / kValueUnit, 0.0f));
        });
      } else {
        // (once: 16320 waves' turns that each did took a millisecond)
        if (lane == 0 && __hip_atomic_load(&p.plan->odd, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) atomicOr(&p.plan->odd, 1);
        store([](float x, float y) { return pack_bf(x, y); });
      }
    } else {
      store([&](float x, float y) { return pack_bf(x, y) ^ p.flip; });
    }
    if (!more) return;
    at = next;
  }
}

__global__ __launch_bounds__(512, 2) void k_prompt_heads(PromptParams p) {
  __shared__ __align__(1024) uint8_t weights[kHalfHead];
  const uint32_t lds = (uint32_t)(uintptr_t)(MKMOE_LDS uint8_t*)&weights[0];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int blocks = uniform(p.plan->rows) / kKeys, halves = 2 * p.heads;
  // The tokens in as many parts as one or eight, and a part's blocks of 64, half head by half head, in equal shares for its
  // workgroups. Eight: an XCD's workgroups go through its part together, and its L2 keeps the tokens between them; one: the
  // shares are evener turns of 8 waves (300 over 65300: 610 and 626 us; ragged prompts' step of 6000 tokens: 205 and 193)
  const int parts = blocks >= 512 ? 8 : 1, groups = gridDim.x / parts;
  const int part = parts == 8 ? blockIdx.x & 7 : 0, me = parts == 8 ? blockIdx.x >> 3 : (blockIdx.x & 7) * (gridDim.x / 8) + (blockIdx.x >> 3);
  const int first = (int)((int64_t)blocks * part / parts), wide = (int)((int64_t)blocks * (part + 1) / parts) - first;
  const int64_t units = (int64_t)wide * halves;
  const int end = (int)(units * (me + 1) / groups);
  for (int unit = (int)(units * me / groups); unit < end;) {
    const int hh = uniform(unit / wide), from = uniform(unit - hh * wide), upto = uniform(min(wide, end - hh * wide));
    if (hh & 1)
      heads_blocks<true>(p, lds, hh >> 1, first + from, first + upto);
    else
      heads_blocks<false>(p, lds, hh >> 1, first + from, first + upto);
    unit = hh * wide + upto;
  }
}

// ---------------------------------------------------------------- attend
// A turn's blocks of 32 keys, W / 4, in LDS: 8 fragments of keys each, then 4 of rope keys each; 8 of values each
constexpr __device__ int blocks_of(int waves) { return waves / 4; }
constexpr __device__ int pe_at(int waves) { return blocks_of(waves) * 8 * kFrag; }
constexpr __device__ int key_lds(int waves) { return blocks_of(waves) * 12 * kFrag; }
constexpr __device__ int val_lds(int waves) { return blocks_of(waves) * 8 * kFrag; }
// turns in LDS: of keys two in use (a block of 32 each), one there or on its way, one requested; of values one less
constexpr int kKeyRing = 4, kValRing = 3;

// a sequence's head's query tile, and the share's part of its keys
struct Item {
  int head, qt;       // qt: of 32 W query rows
  int t0, n, past;    // the sequence's
  int tile;           // its first tile of packed rows; -1: they do not fit, -2: the end of the share
  int tiles;          // turns of keys that the query tile sees
  int from, upto;     // the share's of them
  int parts;          // the shares behind this one that have some, where this one has the first and not all
};
constexpr int kItemWords = sizeof(Item) / 4, kItems = 64;
// item o of the work, for the units begin .. end - 1 of share
__device__ __forceinline__ Item item_of(const PromptParams& p, int o, int share, int begin, int end, int per, int w) {
  Item it{};
  it.tile = -2;
  if (o >= p.plan->items) return it;
  int lo = 0, hi = p.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.plan->item[mid] <= o) lo = mid; else hi = mid - 1;
  }
  const PromptSeq s = prompt_seq(p, lo, p.plan->back != 0);
  const int at = p.plan->at[lo], qts = query_tiles(s.n, w), i = o - p.plan->item[lo];
  it.t0 = s.t0;
  it.n = s.n;
  it.past = s.len - s.n;
  it.head = i / qts;
  it.qt = i - it.head * qts;
  int first = p.plan->work[lo];
  if (at < 0) {
    first += i * kItemSetup;
  } else {
    first += it.head * head_units(it.past, it.n, w) + units_before(it.past, it.qt, w);
    it.tiles = turns_of(it.past, it.n, it.qt, w);
  }
  if (first >= end) return it;
  it.tile = at < 0 ? -1 : at >> 6;
  const int keys = first + kItemSetup;
  it.from = max(0, begin - keys);
  it.upto = min(it.tiles, max(0, end - keys));
  if (it.tiles == 0 && first < begin) it.from = 1;  // (stored by the share that has its first unit)
  it.parts = it.from == 0 && it.upto > 0 && it.upto < it.tiles ? (keys + it.tiles - 1) / per - share : 0;
  return it;
}

// A query row's 32 output values of block vb. The row's two lanes have 4 values of 8 each: they exchange, so that each
// stores 8 that follow each other
__device__ __forceinline__ void store_row(const PromptParams& p, int t0, int n, int head, int row, f32x16 o, int vb, float inv,
                                          int half) {
  uint16_t* to = p.out + (int64_t)(t0 + row) * p.o_ts + (int64_t)head * p.o_hs + 32 * vb + 8 * half;
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    // the first 8 values' words of this lane, the next 8's; then those of half 0's lane are the first 8 values, half 1's the next
    const auto x = __builtin_amdgcn_permlane32_swap(pack_bf(o[i] * inv, o[i + 1] * inv), pack_bf(o[i + 4] * inv, o[i + 5] * inv), false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(pack_bf(o[i + 2] * inv, o[i + 3] * inv), pack_bf(o[i + 6] * inv, o[i + 7] * inv), false, false);
    if (row < n) *(u32x4*)(to + 2 * i) = u32x4{x[0], y[0], x[1], y[1]};
  }
}

// A wave's 32 query rows, a column of lanes each: what they hold while they go through the keys
struct Rows {
  bf16x8 q[12];   // 8 fragments of the values without rotation, dealt, and 4 of the rotated ones
  f32x16 o[4];    // outputs, 32 values each
  float top, mu;  // the largest score so far; what scores times scale log2 e are taken less, kLift below its
  float sum;      // of the lane's numerators
  int sees;       // the last key that the row sees
};
// Numerators are up to 2^(kLift + kMoveBy), below fp16's largest, and what fp16 drops of them is below 2^-32 of the
// largest one's: weights from 2^-24 of the largest have bf16's precision or more, smaller ones less
constexpr float kLift = 7.0f;

// a fragment along a block of 32 keys: 8 of them, then 4 of their rope values
template <int W>
__device__ __forceinline__ uint32_t key_frag(int kb, int ds) {
  return ds < 8 ? (kb * 8 + ds) * kFrag : pe_at(W) + (kb * 4 + ds - 8) * kFrag;
}
// scores of a block of 32 keys: A = keys, B = the queries
template <int W>
__device__ __forceinline__ void score(const Rows& r, f32x16& s, uint32_t at, int kb) {
#pragma unroll
  for (int ds = 0; ds < 12; ++ds) s = mfma32(lds_read<bf16x8>(at + key_frag<W>(kb, ds)), r.q[ds], ds == 0 ? f32x16{} : s);
}
__device__ __forceinline__ void mask_block(const Rows& r, f32x16& s, int key0, int half) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (key0 + 8 * (i >> 2) + 4 * half + (i & 3) > r.sees) s[i] = -__builtin_inff();
}
// Scores times scale log2 e are rounded together with what they are taken less, which differs from the largest one's own
// exponent by its rounding: no more than 2^-13 for exponents up to kFar. Past it (far) scores are taken less the largest one first
constexpr float kFar = 0x1p10f;
// the row's maximum moved to its new scores', where one of the wave's passes it by more than 2^kMoveBy
__device__ __forceinline__ void move_max(const PromptParams& p, Rows& r, bool& far, float top) {
  const auto sw = __builtin_amdgcn_permlane32_swap(f2u(top), f2u(top), false, false);
  top = max3(u2f(sw[0]), u2f(sw[1]), u2f(sw[1]));
  if (__ballot((top - r.top) * p.scale2 > kMoveBy)) {
    const float to = fmaxf(r.top, top), by = to == r.top ? 1.0f : __builtin_amdgcn_exp2f((r.top - to) * p.scale2);
    r.top = to;
    r.mu = to == -__builtin_inff() ? 0.0f : fmaf(to, p.scale2, -kLift);
    far = __ballot(fabsf(r.mu) > kFar) != 0;
    r.sum *= by;
#pragma unroll
    for (int vb = 0; vb < 4; ++vb)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[vb][i] *= by;
  }
}
// log sum exp of a row whose largest score is top
__device__ __forceinline__ float lse_of(const PromptParams& p, float top, float sum) {
  return sum == 0.0f ? -__builtin_inff() : (fmaf(top, p.scale2, -kLift) + __builtin_amdgcn_logf(sum)) * kLog2;
}
__device__ __forceinline__ float top_of(const f32x16& s) {
  float top = s[0];
#pragma unroll
  for (int i = 0; i < 16; i += 2) top = max3(top, s[i], s[i + 1]);
  return top;
}

// The attention. The work is a list of items (a sequence's head's query tile) of units: kItemSetup for an item's start and
// end, and its turns of keys. Every workgroup takes one equal share of the units, whatever the lengths and the causal border
// make of the items; an item that a share's end cuts leaves each wave's fp32 outputs, maxima and sums for
// k_prompt_merge. A wave has 32 query rows, a column of lanes each, and all keys:
//   S^T = K Q^T   A = keys from LDS, B = queries in registers: a lane has 16 scores of its row, so that the row's
//                 maximum takes one exchange with the other half's lane
//   P^T           exp2 of the scores less the maximum, which moves where one passes it by 2^8: fp16, in place
//   O^T += V^T P^T   A = values from LDS, B = P^T as it lies: a row's rescaling is a lane's own factor
// Scores are formed a block of 32 keys ahead, and the code alternates their products with the numerators of the block
// before, then the products of the outputs with the next maximum: a wave's matrix and vector instructions run under
// each other (8191 tokens over 16383 with 32 heads, the call: 2.63 -> 2.03 ms). Keys and values come straight from memory
// to LDS two turns ahead, one barrier a turn. An item's last turn, those whose values are bf16 and those of scores far from 0
// (move_max) go without that, each operand as it is needed: with all values in bf16 the same call takes 2.75 ms, 300 over 65300
// 722 us for 680, ragged prompts' step 224 for 196.
//
// What bounds it: power. 8191 tokens over 16383 with 32 heads, 2.06 PFLOP, take 2.06 ms (the median of 12; 1.98 the least), 1.0
// PFLOP/s (the floor's rate is 1.39): the matrix units are busy for 61 % of the cycles and the clock falls to 1.7 GHz; counters: 3.3
// vector instructions to a matrix instruction, LDS busy for 31 %, without conflicts. Ahead of that, short prompts: an item's
// start and end (its queries, first keys, outputs) of 6 to 9 us beside turns of 1.5 to 2 us of 64 keys.
template <int W>
__global__ __launch_bounds__(64 * W, 2) void k_prompt_attend(PromptParams p) {
  constexpr int NB = blocks_of(W), TK = 32 * NB, kKeyLds = key_lds(W), kValLds = val_lds(W);
  __shared__ __align__(1024) uint8_t ring[kKeyRing * kKeyLds + kValRing * kValLds];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const uint32_t lds = (uint32_t)(uintptr_t)(MKMOE_LDS uint8_t*)&ring[0];
  const uint32_t k_ring = lds, v_ring = lds + kKeyRing * kKeyLds;
  // an XCD's workgroups have shares that follow each other: heads whose keys its L2 keeps
  const int total = uniform(p.plan->total), per = uniform(p.plan->per), shares = (total + per - 1) / per;
  const int by_xcd = (shares + 7) >> 3, share = (blockIdx.x & 7) * by_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= by_xcd || share >= shares) return;
  const int begin = share * per, end = min(total, begin + per);
  const bool any_odd = uniform(p.plan->odd) != 0;
  PromptCut cut{};
  __shared__ int list[kItems][kItemWords];
  int listed = uniform(p.plan->first[share]) - kItems, in_list = kItems;
  // the share's next item (every wave at once: it may fill the list anew)
  auto next_item = [&]() {
    if (in_list == kItems) {
      listed += kItems;
      in_list = 0;
      __syncthreads();
      if (threadIdx.x < kItems) {
        const Item x = item_of(p, listed + threadIdx.x, share, begin, end, per, W);
        int* to = list[threadIdx.x];
        to[0] = x.head, to[1] = x.qt, to[2] = x.t0, to[3] = x.n, to[4] = x.past, to[5] = x.tile, to[6] = x.tiles, to[7] = x.from,
        to[8] = x.upto, to[9] = x.parts;
      }
      __syncthreads();
    }
    const int* x = list[in_list++];
    return Item{uniform(x[0]), uniform(x[1]), uniform(x[2]), uniform(x[3]), uniform(x[4]),
                uniform(x[5]), uniform(x[6]), uniform(x[7]), uniform(x[8]), uniform(x[9])};
  };
  const int64_t kbs = p.cap / 32;

  for (;;) {
    const Item it = next_item();
    if (it.tile == -2) break;
    const int head = it.head, from = it.from, upto = it.upto;
    const int row0 = it.qt * rows_of(W) + wave * 32, row = row0 + col;
    if (from >= upto) {
      if (it.tiles == 0 && from == 0) {
        const float none = it.tile < 0 ? __builtin_nanf("") : 0.0f;
#pragma unroll
        for (int vb = 0; vb < 4; ++vb) store_row(p, it.t0, it.n, head, row, f32x16{} + none, vb, 1.0f, half);
        if (p.lse && half == 0 && row < it.n) p.lse[(int64_t)(it.t0 + row) * p.heads + head] = it.tile < 0 ? none : -__builtin_inff();
      }
      continue;
    }

    const int64_t kb0 = 2 * (int64_t)it.tile;
    // (a wave's fragments; scalar addresses, the lanes 16 bytes apart)
    const uint8_t* kbase = p.k + ((int64_t)head * kbs + kb0) * 8 * kFrag + wave * 2 * kFrag;
    const uint8_t* vbase = p.v + ((int64_t)head * kbs + kb0) * 8 * kFrag + wave * 2 * kFrag;
    const uint8_t* pbase = p.pe + kb0 * 4 * kFrag + wave * kFrag;
    auto issue_k = [&](int kt) {
      const uint32_t to = k_ring + (kt % kKeyRing) * kKeyLds;
      const uint8_t* from_k = kbase + (int64_t)kt * NB * 8 * kFrag;
      lds_dma16(from_k, lane * 16, to + wave * 2 * kFrag);
      lds_dma16(from_k + kFrag, lane * 16, to + wave * 2 * kFrag + kFrag);
      lds_dma16(pbase + (int64_t)kt * NB * 4 * kFrag, lane * 16, to + pe_at(W) + wave * kFrag);
    };
    auto issue_v = [&](int kt) {
      const uint32_t to = v_ring + (kt % kValRing) * kValLds + wave * 2 * kFrag;
      const uint8_t* from_v = vbase + (int64_t)kt * NB * 8 * kFrag;
      lds_dma16(from_v, lane * 16, to);
      lds_dma16(from_v + kFrag, lane * 16, to + kFrag);
    };

    Rows r;
    {
      const uint16_t* qn = p.qn + (int64_t)(it.t0 + row) * p.qn_ts + (int64_t)head * p.qn_hs + 4 * half;
      const uint16_t* qp = p.qp + (int64_t)(it.t0 + row) * p.qp_ts + (int64_t)head * p.qp_hs + 8 * half;
#pragma unroll
      for (int ds = 0; ds < 12; ++ds) r.q[ds] = bf16x8{};
      if (row < it.n) {  // (the other columns reach nothing)
#pragma unroll
        for (int ds = 0; ds < 8; ++ds) {
          const u32x2 a = *(const u32x2*)(qn + 16 * ds), b = *(const u32x2*)(qn + 16 * ds + 8);
          r.q[ds] = __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
        }
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) r.q[8 + ds] = *(const bf16x8*)(qp + 16 * ds);
      }
    }
    // of 64 turns from marks_from on, those whose values are bf16, and those of them with some that may not be finite
    const int32_t* odd = p.odd + (int64_t)head * (p.cap / kKeys) + it.tile;
    uint64_t marked = 0, not_finite = 0;
    int marks_from = from;
    auto read_marks = [&](int kt) {
      const int mark = kt + lane < upto ? odd[(kt + lane) * TK / kKeys] : 0;
      marked = __ballot(mark != 0);
      not_finite = __ballot(mark == 2);
      marks_from = kt;
    };
    if (any_odd) read_marks(from);
    barrier();  // every wave has read the turns of the item before

    r.top = -__builtin_inff();
    r.mu = r.sum = 0.0f;
    r.sees = it.past + row;  // the last key that the row sees
#pragma unroll
    for (int vb = 0; vb < 4; ++vb) r.o[vb] = f32x16{};
    // the tiles that the wave's rows see, and those that all of them see whole
    const int last_row = min(row0 + 31, it.n - 1);
    const int seen = row0 < it.n ? min(upto, (it.past + last_row + TK) >> key_shift(W)) : from;
    const int whole = (it.past + row0 + 1) >> key_shift(W);

    issue_k(from);
    if (from + 1 < upto) issue_k(from + 1);
    issue_v(from);
    if (from + 2 < upto) issue_k(from + 2);
    if (from + 1 < upto) issue_v(from + 1);
    // at turn kt the keys of kt + 1 and the values of kt are there; the next turn's are on their way
    auto turn = [&](int kt) {
      if (kt + 2 < upto)
        wait_loads<5>();
      else
        wait_loads<0>();
      barrier();
      if (kt + 3 < upto) issue_k(kt + 3);
      if (kt + 2 < upto) issue_v(kt + 2);
    };
    auto keys_at = [&](int kt) { return k_ring + (kt % kKeyRing) * kKeyLds + lane * 16; };
    auto vals_at = [&](int kt) { return v_ring + (kt % kValRing) * kValLds + lane * 16; };
    // a block of 32 keys' scores are formed one block ahead: its numerators then come under the next one's products
    f32x16 s0, s1;
    if (from + 2 < upto)
      wait_loads<10>();
    else
      wait_loads<0>();
    barrier();
    int kt = from;
    bool far = false;  // some row's scores are
    if (seen > from) {
      score<W>(r, s0, keys_at(from), 0);
      if (from >= whole) mask_block(r, s0, from * TK, half);
      move_max(p, r, far, top_of(s0));
    }
    while (kt < upto) {
      int plain = upto;  // the turns before it have values in fp16
      if (any_odd) {
        if (kt - marks_from >= 63) read_marks(kt);
        const uint64_t ahead = marked >> (kt - marks_from);
        plain = ahead != 0 ? kt + __builtin_ctzll(ahead) : marks_from + 63;
      }
      // two blocks a time, of one turn or of two, as long as there is a block behind them
      const int fast = min(seen, plain + 1);
      bool swapped = false;
      while (!far && !swapped && kt + 1 < fast) {
        turn(kt);
        uint32_t k_at = keys_at(NB == 2 ? kt : kt + 1), v_at = vals_at(kt), next_at = keys_at(kt + 1);
        // 20 fragments a block in turn: 12 of keys for the next block's scores, 8 of values for this one's outputs; each
        // is read two products before its own
        u32x4 f[3], num[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if (hh == 1) {
            if (NB == 1) ++kt;
            swapped = far || (NB == 1 && kt + 1 >= fast);
            if (swapped) break;
            if (NB == 1) {
              turn(kt);
              next_at = keys_at(kt + 1);
              v_at = vals_at(kt);
            }
          }
          f32x16 &now = hh == 0 ? s0 : s1, &then = hh == 0 ? s1 : s0;
          auto frag = [&](int j) {
            return lds_read<u32x4>(j >= 12  ? v_at + ((NB == 2 ? hh * 8 : 0) + j - 12) * kFrag
                                   : hh == 0 ? k_at + key_frag<W>(NB - 1, j)
                                             : next_at + key_frag<W>(0, j));
          };
          f[0] = frag(0);
          f[1] = frag(1);
#pragma unroll
          for (int j = 0; j < 12; ++j) {
            f[(j + 2) % 3] = frag(j + 2);
            then = mfma32(__builtin_bit_cast(bf16x8, f[j % 3]), r.q[j], j == 0 ? f32x16{} : then);
#pragma unroll
            for (int x = j * 8 / 12; x < (j + 1) * 8 / 12; ++x) {
              uint32_t w = pack_f16(__builtin_amdgcn_exp2f(now[2 * x] * p.scale2 - r.mu),
                                    __builtin_amdgcn_exp2f(now[2 * x + 1] * p.scale2 - r.mu));
              r.sum = add_f16(w, r.sum);
              asm volatile("" : "+v"(w), "+v"(r.sum));  // (formed here, not where they are used)
              num[x >> 2][x & 3] = w;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          // the next block's turn and first key
          const int next_kt = NB == 2 ? kt + hh : kt + 1, key0 = NB == 2 ? kt * TK + (hh + 1) * 32 : (kt + 1) * TK;
          float top = -__builtin_inff();
#pragma unroll
          for (int j = 12; j < 20; ++j) {
            const int vb = j & 3;
            if (j + 2 < 20) f[(j + 2) % 3] = frag(j + 2);
            r.o[vb] = mfma32(__builtin_bit_cast(f16x8, f[j % 3]), __builtin_bit_cast(f16x8, num[(j - 12) >> 2]), r.o[vb]);
            if (j == 14 && next_kt >= whole) mask_block(r, then, key0, half);
            if (j >= 14) {
#pragma unroll
              for (int x = (j - 14) * 8 / 6; x < (j - 13) * 8 / 6; ++x) top = max3(top, then[2 * x], then[2 * x + 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          move_max(p, r, far, top);
        }
        if (!swapped) ++kt;
      }
      // a turn of any kind
      int done = 0;  // blocks of it that are
      if (swapped) {
        s0 = s1;
        done = NB - 1;
      }
      if (done == 0) turn(kt);
      if (kt < seen) {
        const bool in_bf = any_odd && (marked >> (kt - marks_from) & 1) != 0;
#pragma unroll
        for (int hh = 0; hh < NB; ++hh) {
          if (hh < done) continue;
          const uint32_t v_at = vals_at(kt) + hh * 8 * kFrag;
          const float top = r.top == -__builtin_inff() ? 0.0f : r.top, lift = in_bf ? kLift + kValueLift : kLift;
          u32x4 num[2];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float y = __builtin_amdgcn_exp2f(fmaf(s0[2 * x] - top, p.scale2, lift));
            const float z = __builtin_amdgcn_exp2f(fmaf(s0[2 * x + 1] - top, p.scale2, lift));
            const uint32_t w = in_bf ? pack_bf(y, z) : pack_f16(y, z);
            r.sum = in_bf ? add_bf16(w, r.sum) : add_f16(w, r.sum);
            num[x >> 2][x & 3] = w;
          }
          if (in_bf && kt >= whole && (not_finite >> (kt - marks_from) & 1) != 0) {
            // values that may not be finite, of tokens that some rows do not see: a key at a time, added where it is seen
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int vb = 0; vb < 4; ++vb)
#pragma unroll 1
                for (int x = 0; x < 16; ++x) {
                  const int h = x >> 3, e = x & 7;
                  const bool sees = kt * TK + 32 * hh + 16 * t + 8 * (e >> 2) + 4 * h + (e & 3) <= r.sees;
                  const uint32_t word = half == h ? (e & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
                  const u32x4 only = {e >> 1 == 0 ? word : 0u, e >> 1 == 1 ? word : 0u, e >> 1 == 2 ? word : 0u, e >> 1 == 3 ? word : 0u};
                  const u32x4 a = lds_read<u32x4>(v_at + (t * 4 + vb) * kFrag);
                  const f32x16 add = mfma32(__builtin_bit_cast(bf16x8, a & only), __builtin_bit_cast(bf16x8, num[t] & only), f32x16{});
#pragma unroll
                  for (int i = 0; i < 16; ++i) r.o[vb][i] += sees ? add[i] : 0.0f;
                }
          } else if (in_bf) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              r.o[j & 3] = mfma32(lds_read<bf16x8>(v_at + j * kFrag), __builtin_bit_cast(bf16x8, num[j >> 2]), r.o[j & 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              r.o[j & 3] = mfma32(lds_read<f16x8>(v_at + j * kFrag), __builtin_bit_cast(f16x8, num[j >> 2]), r.o[j & 3]);
          }
          const int then = kt + (hh + 1) / NB;  // the next block's turn
          if (then < seen) {
            score<W>(r, s0, keys_at(then), (hh + 1) % NB);
            if (then >= whole) mask_block(r, s0, kt * TK + (hh + 1) * 32, half);
            move_max(p, r, far, top_of(s0));
          }
        }
      }
      s1 = f32x16{};  // (it is formed anew: without that, registers were kept for it)
      ++kt;
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(f2u(r.sum), f2u(r.sum), false, false);
    const float sum = u2f(sw[0]) + u2f(sw[1]);
    if (from == 0 && upto == it.tiles) {
      const float inv = sum == 0.0f ? 0.0f : kValueUnit / sum;
#pragma unroll
      for (int vb = 0; vb < 4; ++vb) store_row(p, it.t0, it.n, head, row, r.o[vb], vb, inv, half);
      if (p.lse && half == 0 && row < it.n)
        p.lse[(int64_t)(it.t0 + row) * p.heads + head] = lse_of(p, r.top, sum);
    } else if (row0 < it.n) {
      const int slot = 2 * share + (from == 0);
      f32x4* to = (f32x4*)p.part_o + ((int64_t)slot * W + wave) * 16 * 64 + lane;
#pragma unroll
      for (int vb = 0; vb < 4; ++vb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          to[(vb * 4 + i) * 64] = f32x4{r.o[vb][4 * i], r.o[vb][4 * i + 1], r.o[vb][4 * i + 2], r.o[vb][4 * i + 3]};
      // (where the row saw no score yet its largest is -inf, its sum 0, and the part counts for nothing)
      if (half == 0) *(f32x2*)(p.part_ml + ((int64_t)slot * rows_of(W) + wave * 32 + col) * 2) = f32x2{r.top, sum};
    }
    if (it.parts > 0) cut = PromptCut{it.parts, it.head, it.t0, it.n, it.qt, {}};
  }
  if (threadIdx.x == 0 && cut.parts > 0) p.cut[share] = cut;
}

// The parts of query tiles that the ends of shares cut, joined: of a tile 32 rows a workgroup and turn, 32 values of them
// and every fourth part a wave, so that a tile of many parts (few heads over long keys) has its loads on their way at once. The
// four waves' sums are joined in order. The lanes have the values that the attention's had. Every workgroup lists the
// cut tiles itself: a workgroup for each share and rows, most of them for nothing, took 6 us to launch.
template <int W>
__global__ __launch_bounds__(1024, 8) void k_prompt_merge(PromptParams p) {
  __shared__ f32x4 sums[3][4][4][64];
  __shared__ f32x2 tops[3][4][64];
  __shared__ int list[kMaxShares][6], counts[kMaxShares / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, vb = wave & 3, slice = wave >> 2;
  const int half = lane >> 5, col = lane & 31;
  PromptCut mine{};
  if (tid < shares_of(W)) mine = p.cut[tid];
  const uint64_t those = __ballot(mine.parts > 0);
  if (lane == 0 && wave < kMaxShares / 64) counts[wave] = __builtin_popcountll(those);
  __syncthreads();
  int before = 0, cuts = 0;
#pragma unroll
  for (int i = 0; i < kMaxShares / 64; ++i) {
    if (i < wave) before += counts[i];
    cuts += counts[i];
  }
  if (mine.parts > 0) {
    int* to = list[before + __builtin_popcountll(those & ((1ull << lane) - 1))];
    to[0] = mine.parts, to[1] = mine.head, to[2] = mine.t0, to[3] = mine.n, to[4] = mine.qt, to[5] = tid;
  }
  for (int job = blockIdx.x; job < cuts * W; job += gridDim.x) {
    __syncthreads();  // (the list is there; the sums before have been read)
    const int* from = list[job / W];
    const PromptCut c = {uniform(from[0]), uniform(from[1]), uniform(from[2]), uniform(from[3]), uniform(from[4]), {}};
    const int share = uniform(from[5]), group = job % W;
    const int row0 = c.qt * rows_of(W) + group * 32, row = row0 + col;
    if (row0 >= c.n) continue;
    auto slot = [&](int i) { return 2 * (share + i) + (i == 0); };
    auto ml_of = [&](int i) { return *(const f32x2*)(p.part_ml + ((int64_t)slot(i) * rows_of(W) + group * 32 + col) * 2); };
    auto part_of = [&](int i, f32x4 (&x)[4]) {
      const f32x4* from = (const f32x4*)p.part_o + (((int64_t)slot(i) * W + group) * 16 + vb * 4) * 64 + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = from[j * 64];
    };
    f32x16 o = {};
    float sum = 0.0f, top = -__builtin_inff();
    auto add = [&](f32x2 ml, const f32x4 (&x)[4]) {
      const float by = ml[0] == top ? 1.0f : __builtin_amdgcn_exp2f((ml[0] - top) * p.scale2);
      sum += ml[1] * by;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] += x[i >> 2][i & 3] * by;
    };
    if (slice <= c.parts) {
      f32x4 x[4];
      const f32x2 ml = ml_of(slice);
      part_of(slice, x);  // (on its way while the maximum is found)
      top = ml[0];
#pragma unroll 8
      for (int i = slice + 4; i <= c.parts; i += 4) top = fmaxf(top, ml_of(i)[0]);
      add(ml, x);
#pragma unroll 2
      for (int i = slice + 4; i <= c.parts; i += 4) {
        part_of(i, x);
        add(ml_of(i), x);
      }
    }
    if (slice > 0 && slice <= c.parts) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[slice - 1][vb][j][lane] = f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
      tops[slice - 1][vb][lane] = f32x2{top, sum};
    }
    __syncthreads();
    if (slice > 0) continue;
    const int more = min(c.parts, 3);
    float all = top;
    for (int i = 0; i < more; ++i) all = fmaxf(all, tops[i][vb][lane][0]);
    const float by0 = top == all ? 1.0f : __builtin_amdgcn_exp2f((top - all) * p.scale2);
    sum *= by0;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= by0;
    for (int i = 0; i < more; ++i) {
      const f32x2 ml = tops[i][vb][lane];
      const float by = ml[0] == all ? 1.0f : __builtin_amdgcn_exp2f((ml[0] - all) * p.scale2);
      sum += ml[1] * by;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 x = sums[i][vb][j][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * j + e] += x[e] * by;
      }
    }
    store_row(p, c.t0, c.n, c.head, row, o, vb, sum == 0.0f ? 0.0f : kValueUnit / sum, half);
    if (p.lse && vb == 0 && half == 0 && row < c.n)
      p.lse[(int64_t)(c.t0 + row) * p.heads + c.head] = lse_of(p, all, sum);
  }
}

// ---------------------------------------------------------------- host
// a workspace: the latent calls' own first (its error words serve both), then the prompt's
struct PromptLayout {
  size_t plan, cut, part_ml, part_o, odd, pe, c, k, v, bytes;
};
inline PromptLayout prompt_layout(int heads, int64_t cap) {
  PromptLayout l;
  size_t at = 0;
  (void)mkmoe_latent_workspace_bytes(&at);
  auto take = [&](size_t n) {
    const size_t from = at;
    at += (n + 255) & ~(size_t)255;
    return from;
  };
  l.plan = take(sizeof(Plan));
  l.cut = take(kMaxShares * sizeof(PromptCut));
  l.part_ml = take((size_t)2 * 2048 * 32 * 2 * 4);
  l.part_o = take((size_t)2 * 2048 * 32 * kV * 4);
  l.odd = take((size_t)heads * (cap / kKeys) * 4);
  l.pe = take((size_t)cap * kR * 2);
  l.c = take((size_t)cap * kL * 2);
  l.k = take((size_t)heads * cap * kNope * 2);
  l.v = take((size_t)heads * cap * kV * 2);
  l.bytes = at;
  return l;
}
constexpr int kMaxContext = 1 << 22, kMaxPromptTokens = 1 << 20;
inline int prompt_params(const mkmoe_latent_prompt_io* io, void* ws, size_t ws_bytes, PromptParams& p) {
  if (!io || !ws) return MKMOE_ERR_NULL;
  if (!aligned(ws, 256)) return MKMOE_ERR_ALIGN;
  if (int rc = check_cache(io->cache)) return rc;
  if (!io->q_nope || !io->q_pe || !io->w || !io->table || !io->lens || !io->out) return MKMOE_ERR_NULL;
  if (io->seqs < 1 || io->seqs > kPromptSeqs || io->tokens < 0 || io->tokens > kMaxPromptTokens) return MKMOE_ERR_ROWS;
  if (!io->q_starts && io->tokens % io->seqs != 0) return MKMOE_ERR_ROWS;
  if (io->heads < 1 || io->heads > MKMOE_LATENT_MAX_HEADS || io->max_context < 1 || io->max_context > kMaxContext)
    return MKMOE_ERR_ARG;
  const int64_t cap = packed_rows(io->max_context);
  const PromptLayout l = prompt_layout(io->heads, cap);
  if (ws_bytes < l.bytes) return MKMOE_ERR_WORKSPACE;
  const float scale2 = fabsf(io->scale) * kLog2E;
  if (!isfinite(scale2) || io->max_pages < 1 || io->table_stride < io->max_pages) return MKMOE_ERR_ARG;
  const int64_t max_len = (int64_t)io->max_pages * io->cache.page_size;
  if (max_len > (int64_t)1 << 30) return MKMOE_ERR_ARG;
  p.waves = prompt_waves(*io);
  if (p.waves == 0) return MKMOE_ERR_ARG;
  const void* wide[] = {io->q_nope, io->q_pe, io->w, io->out};
  for (const void* q : wide)
    if (!aligned(q, 16)) return MKMOE_ERR_ALIGN;
  const void* narrow[] = {io->table, io->lens, io->q_starts, io->lse};
  for (const void* q : narrow)
    if (!aligned(q, 4)) return MKMOE_ERR_ALIGN;
  if (!strides8(io->qn_token_stride, io->qn_head_stride) || !strides8(io->qp_token_stride, io->qp_head_stride) ||
      !strides8(io->out_token_stride, io->out_head_stride))
    return MKMOE_ERR_ALIGN;
  if (!rows_apart(io->out_token_stride, io->tokens, io->out_head_stride, io->heads, kV)) return MKMOE_ERR_ARG;
  uint8_t* at = (uint8_t*)ws;
  p.qn = (const uint16_t*)io->q_nope;
  p.qp = (const uint16_t*)io->q_pe;
  p.w = (const uint16_t*)io->w;
  p.cache = (const uint8_t*)io->cache.data;
  p.table = io->table;
  p.lens = io->lens;
  p.starts = io->q_starts;
  p.out = (uint16_t*)io->out;
  p.lse = io->lse;
  p.err = (int32_t*)at;
  p.plan = (Plan*)(at + l.plan);
  p.cut = (PromptCut*)(at + l.cut);
  p.part_ml = (float*)(at + l.part_ml);
  p.part_o = (float*)(at + l.part_o);
  p.odd = (int32_t*)(at + l.odd);
  p.pe = at + l.pe;
  p.c = at + l.c;
  p.k = at + l.k;
  p.v = at + l.v;
  p.qn_ts = io->qn_token_stride;
  p.qn_hs = io->qn_head_stride;
  p.qp_ts = io->qp_token_stride;
  p.qp_hs = io->qp_head_stride;
  p.o_ts = io->out_token_stride;
  p.o_hs = io->out_head_stride;
  p.table_stride = io->table_stride;
  p.cap = cap;
  p.pages = (int)io->cache.pages;
  p.seqs = io->seqs;
  p.tokens = io->tokens;
  p.heads = io->heads;
  p.n = io->q_starts ? 0 : io->tokens / io->seqs;
  p.max_len = (int)max_len;
  p.page_shift = __builtin_ctz((unsigned)io->cache.page_size);
  // (a scale of 0 weighs every visible token alike; the masked ones' infinities need a factor above 0)
  p.scale2 = fmaxf(scale2, 0x1p-126f);
  p.flip = io->scale < 0.0f ? 0x80008000u : 0u;
  return MKMOE_OK;
}

template <int W>
int attend_and_merge(const PromptParams& p, hipStream_t st) {
  hipLaunchKernelGGL(k_prompt_attend<W>, dim3(shares_of(W)), dim3(64 * W), 0, st, p);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(k_prompt_merge<W>, dim3(512), dim3(1024), 0, st, p);
  return launched();
}
inline int prompt_launch(const PromptParams& p, bool mx, hipStream_t st) {
  const int64_t rows = p.cap < (int64_t)p.seqs * p.max_len ? p.cap : (int64_t)p.seqs * p.max_len;
  const int64_t blocks = (rows + 31) / 32 + p.seqs;
  const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024) + 1);  // (and the planner)
  if (mx)
    hipLaunchKernelGGL(k_prompt_rows<true>, grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(k_prompt_rows<false>, grid, dim3(256), 0, st, p);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(k_prompt_heads, dim3(256), dim3(512), 0, st, p);
  if (int rc = launched()) return rc;
  return p.waves == 8 ? attend_and_merge<8>(p, st) : attend_and_merge<4>(p, st);
}

}  // namespace mkmoe_latent

extern "C" {

int mkmoe_latent_prompt_bytes(int32_t heads, int32_t max_context, size_t* bytes) {
  using namespace mkmoe_latent;
  if (!bytes) return MKMOE_ERR_NULL;
  if (heads < 1 || heads > MKMOE_LATENT_MAX_HEADS || max_context < 1 || max_context > kMaxContext) return MKMOE_ERR_ARG;
  *bytes = prompt_layout(heads, packed_rows(max_context)).bytes;
  return MKMOE_OK;
}

int mkmoe_latent_prompt(const mkmoe_latent_prompt_io* io, void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  PromptParams p;
  if (int rc = prompt_params(io, ws, ws_bytes, p)) return rc;
  if (p.tokens == 0) return MKMOE_OK;
  return prompt_launch(p, io->cache.fmt == MKMOE_LATENT_MXFP8, (hipStream_t)stream);
}

int mkmoe_latent_prompt_step(const mkmoe_latent_append_io* append, const mkmoe_latent_prompt_io* io, void* ws,
                             size_t ws_bytes, void* stream) {
  using namespace mkmoe_latent;
  PromptParams p;
  if (int rc = prompt_params(io, ws, ws_bytes, p)) return rc;
  if (!append) return MKMOE_ERR_NULL;
  if (append->tokens != io->tokens) return MKMOE_ERR_ROWS;
  const mkmoe_latent_cache &from = append->cache, &to = io->cache;
  if ((append->heads != 0 && append->heads != io->heads) || from.data != to.data || from.pages != to.pages ||
      from.page_size != to.page_size || from.fmt != to.fmt)
    return MKMOE_ERR_ARG;
  // (it checks its own arguments before it launches)
  if (int rc = append_for_step(append, ws, ws_bytes, (hipStream_t)stream)) return rc;
  if (p.tokens == 0) return MKMOE_OK;
  return prompt_launch(p, io->cache.fmt == MKMOE_LATENT_MXFP8, (hipStream_t)stream);
}

}  // extern "C"
