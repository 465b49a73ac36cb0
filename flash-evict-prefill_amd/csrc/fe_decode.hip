// Attention of new tokens over a bounded KV cache, and the replay of the weights they gave it, for gfx950.
//
// For batch row b and KV head j (query heads g = 0 .. G-1 of the group, n = length[b, j] cache rows, T new
// tokens), with x = scale * q . k over the n cache rows and the new rows u that tree[t, u] shows to query t
// (u <= t without a tree):
//
//   lse[g, t] = log sum exp x        p = exp(x - lse)        out[g, t] = sum p * value
//   importance_out[s] = importance[s] * exp(-decay * A) + norm[s] * sum_{g, i} w_i p[g, i, s]
//   new_importance[u] = |v_u|_1 * sum_{g, i} w_i p[g, i, u]          w_i = exp(-decay * (A - 1 - i))
//
// where the rows i are the A new tokens that stay: all T of a chunk, or the accepted path of a drafted tree.
// Counting recency back from the newest token, a prompt's importance continued chunk by chunk is the
// importance of the whole (fe_prefill's).
//
//   decode_few_kernel      up to 16 query rows r = g * T + t of a group, the steps of one or a few tokens: each wave takes
//                          32 keys at a time for all of them, S^T = K Q^T and O^T = V^T P^T on MFMA, with the rows' running
//                          maximum and sum
//   decode_wide_kernel     more rows: each wave holds 32 of them, the block's waves share tiles of 64 keys in LDS
//   decode_elements_kernel any layout of rows that 16-byte loads cannot read
//   decode_join_kernel     joins the splits of the keys: out and lse; and, where the first kernel left its logits
//                          (few rows), the importance, whose probabilities need the joined lse
//   decode_replay_kernel   the importance otherwise: S = Q K^T for the rows that stay, lanes holding keys, so that a
//                          key's sum over the rows is in-lane: w p = exp2((x - lse) log2e + log2 w); the difference is
//                          taken in lse's own units, where it rounds once
//                          (decode_replay_elements_kernel for rows that do not allow 16-byte loads)
//
// Sums, maxima and partial outputs are FP32. Probabilities are rounded to the inputs' type, as the second product takes
// them: half a step of each, which the output's own rounding has too; outputs are normalised by the sum of the rounded
// ones. lse and the importance take the exact ones.
//
// Lengths are known on the device only: a launch's grid comes from the cache's size, and a head's blocks divide the
// tiles that its length has, or all heads' blocks all tiles (dec_assign).
// Short calls are bound by code that runs for the first time and by trips to memory one after the other. So registers
// do not spill, the loads of a tile are in the code once, rows past the end are read as the last, arguments are read at
// once (dec_hold), and little is divided: the first version of this file, which did none of that, took 15.4 + 11.0 us
// for a step over 1024 rows of 8 heads, against 6.1 + 5.3 us.
#include <math.h>
#include <stddef.h>
#include <algorithm>
#include <string>

#include "fe_attn.h"
#include "fe_internal.h"
#include "fe_radix.h"
#include "../../include/flash_evict.h"

namespace fe {

typedef __attribute__((address_space(3))) void* dec_lds_ptr;
typedef short dec_s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) dec_s16x4 dec_lds_s16x4;

constexpr int kDecMaxTokens = 256;   // new tokens of a call
// Rows of a group up to which decode_few_kernel takes them: it has one tile of 16. With a second one it took 11.3 us for
// 32 rows of 8 heads over 1024 rows of the cache and 38.5 us of 32 heads over 8192, the wide kernel 12.4 and 31.2.
constexpr int kDecFewRows = 16;
// Rows of a group up to which the attention leaves its logits for the importance: 8 bytes a row and key, written and
// read, against the 2 D of reading K again. Measured with the logits and without, 8 heads: 4 rows over 131072 keys 123
// and 164 us, over 1024 11.5 and 13.9; 16 rows over 65536 65 and 74.
constexpr int kDecLogitRows = 16;
// Blocks that share the importance of all heads: a step over 131072 rows 128.7 us with 256, 123 with 1024, 128 with 4096.
constexpr int kDecJoinBlocks = 1024;
// Pointers to global memory, said to be: a pointer that the compiler loses sight of (dec_hold) would be read with flat
// instructions, which wait for LDS too.
#define FE_GLOBAL __attribute__((address_space(1)))
typedef const FE_GLOBAL u16* DecIn;
typedef FE_GLOBAL float* DecF32;
typedef const FE_GLOBAL float* DecF32In;
typedef const FE_GLOBAL int* DecI32In;

// Attention. Slots: ((b * Hkv + j) * RB + row block) * S + split; of the wide kernel and where heads share the blocks, block *
// RB + row block, with a head's first block and their number in `heads`.
struct DecArgs {
  DecIn q, k, v, kc, vc;   // queries, new rows, the cache
  DecI32In length;         // [B * Hkv]
  const FE_GLOBAL unsigned char* tree;   // [T, T] or [B, T, T], or null: causal
  DecF32 part_o;           // [slot][RS][DP]: normalised partial outputs
  DecF32 part_ml;          // [slot][2][RS]: maximum (log2 units), sum
  DecF32 logits;           // [B * Hkv][tile of 32 keys][R][32] in log2 units, or null
  long long qb, qh, qn, kb, kh, vb, vh, kcb, kch, vcb, vch, tree_stride;   // strides of batch, head, (q) row
  u32 kn, vn, kcn, vcn;    // row strides
  int T, C, D, R, RB, RS, S, max_tiles;   // R rows of a group in RB blocks of RS; splits; tiles of a full cache
  u32 qand, qxor;          // Q's sign for a negative scale, Q's zeros for a zero one
  float scale_log2;
  int Hkv, BH, NB;         // BH: all heads; NB: blocks they share, or 0
  FE_GLOBAL int* heads;    // [B * Hkv][2]
  int pad[2];
  // element loads: 64-bit row strides, channel strides
  long long kn64, vn64, kcn64, vcn64, qc, kd, vd, kcd, vcd;
};
static_assert(offsetof(DecArgs, pad) <= 4 * 64 && sizeof(DecArgs) >= 4 * 64, "argument window");

struct DecReplayArgs {
  DecIn q, k, v, kc;
  DecI32In length, path;   // path: or null, all T
  DecF32In lse, imp, norm;
  DecF32 imp_out, new_imp;
  long long qb, qh, qn, kb, kh, vb, vh, kcb, kch;   // strides of batch, head, (q) row
  long long imp_stride, norm_stride, impo_stride;
  u32 kn, vn, kcn;         // row strides
  int T, C, D, G, A, S;
  float scale, decay_log2;
  int Hkv, BH, NB;         // as above
  int pad[5];
  // element loads: 64-bit row strides, channel strides
  long long kn64, vn64, kcn64, qc, kd, vd, kcd;
};
static_assert(offsetof(DecReplayArgs, pad) <= 4 * 64 && sizeof(DecReplayArgs) >= 4 * 64, "argument window");

struct DecJoinArgs {
  DecF32In part_o, part_ml, logits;
  DecI32In length, heads;  // heads: as above, or null
  FE_GLOBAL u16* out;      // [B, Hq, T, D]
  DecF32 lse;              // [B, Hq, T]
  DecF32In imp, norm;
  DecF32 imp_out, new_imp;
  DecIn v;
  long long imp_stride, norm_stride, impo_stride, vb, vh, vn, vd;
  int T, C, D, R, RB, RS, S, max_tiles;
  int rows;                // output rows of a block: 1, all its threads on it, or a group of threads on each
  int out_blocks;          // of a head
  float decay_log2;
  int pad[15];
};
static_assert(offsetof(DecJoinArgs, pad) <= 4 * 64 && sizeof(DecJoinArgs) >= 4 * 64, "argument window");

// The kernel's arguments, the first 256 bytes of them read at once and kept in registers. Left to the compiler, each is read
// where it is first used and again wherever that saves registers, with a wait each time.
template <typename A>
__device__ __forceinline__ A dec_hold(const A& arg) {
  static_assert(sizeof(A) >= 4 * 64, "argument window");
  A a = arg;
  typedef u32 u32x16 __attribute__((ext_vector_type(16), aligned(4)));
  typedef const __attribute__((address_space(4))) u32x16* args_ptr;
  const args_ptr p = (args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
  u32x16 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = p[i];
  asm volatile("" : "+s"(v[0]), "+s"(v[1]), "+s"(v[2]), "+s"(v[3]));
  // from here on word by word: a spilled register of 16 words would come back whole for each word of it
  u32 w[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    w[i] = v[i / 16][i % 16];
    asm volatile("" : "+s"(w[i]));
  }
  __builtin_memcpy((char*)&a, w, 4 * 64);
  return a;
}

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kDecNegInf = -__builtin_huge_valf();

// Orders a wave's own LDS writes and reads (the hardware keeps them in order; the compiler is told).
__device__ __forceinline__ void dec_wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Rows of DP 16-bit channels in LDS, in order, with their 16-byte chunks permuted. K: the fragment reads take one
// chunk of 16 consecutive rows in a phase; the permutation puts these on all 64 banks. V: a transposing read takes
// 64 bytes of four consecutive rows; their 64-byte groups are permuted likewise.
template <int DP>
__device__ __forceinline__ int dec_kswz(int row) {
  return DP % 128 == 0 ? row & 15 : (DP % 64 == 0 ? (row >> 1) & 7 : (row >> 2) & 3);
}
template <int DP>
__device__ __forceinline__ int dec_k_at(int row, int chunk) { return (row * (DP / 8) + (chunk ^ dec_kswz<DP>(row))) * 16; }
template <int DP>
__device__ __forceinline__ int dec_vswz(int row) {
  return DP % 128 == 0 ? row & 3 : (DP % 64 == 0 ? (row >> 1) & 1 : 0);
}
template <int DP>
__device__ __forceinline__ int dec_v_at(int row, int chunk) {
  return row * (DP * 2) + ((chunk >> 2) ^ dec_vswz<DP>(row)) * 64 + (chunk & 3) * 16;
}
// K fragment c (16 channels) of rows r0 + l32
template <int DP>
__device__ __forceinline__ u32x4 dec_kfrag(const unsigned char* kt, int r0, int c) {
  const int l32 = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1;
  return *(const u32x4*)(kt + dec_k_at<DP>(r0 + l32, 2 * c + hh));
}
// V^T fragment of channels 32 dt .. + 31, keys r0 .. r0 + 15: eight keys of channel 32 dt + l32 a lane, in the order of
// the S^T accumulators (r0 + 4 hh + 0..3, then r0 + 8 + 4 hh + 0..3)
template <int DP>
__device__ __forceinline__ u32x4 dec_vfrag(unsigned char* vt, int r0, int dt) {
  const int lane = threadIdx.x & 63, tr = lane & 15, tg = lane >> 4, hh = lane >> 5;
  const int row = r0 + 4 * hh + (tr >> 2);
  unsigned char* p = vt + row * (DP * 2) + (dt ^ dec_vswz<DP>(row)) * 64 + 32 * (tg & 1) + 8 * (tr & 3);
  // row + 8 has the same permutation
  const u32x2 ux = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)p));
  const u32x2 uy = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)(p + 8 * DP * 2)));
  return (u32x4){ux[0], ux[1], uy[0], uy[1]};
}

// 16 bytes of a row: channels 8 ch .. 8 ch + 7, zeros past D.
__device__ __forceinline__ u32x4 dec_load8(DecIn row, long long cs, int ch, int D) {
  u32 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int da = 8 * ch + 2 * i, db = da + 1;
    const u32 lo = da < D ? (u32)row[da * cs] : 0u, hi = db < D ? (u32)row[db * cs] : 0u;
    w[i] = lo | (hi << 16);
  }
  return (u32x4){w[0], w[1], w[2], w[3]};
}

// Whether one of eight 16-bit values is an infinity or a NaN.
template <typename E>
__device__ __forceinline__ bool dec_nonfinite(u32x4 x);
template <u32 MASK>
__device__ __forceinline__ bool dec_exponent_full(u32x4 x) {
  bool bad = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) bad |= (x[w] & MASK) == MASK || ((x[w] >> 16) & MASK) == MASK;
  return bad;
}
template <>
__device__ __forceinline__ bool dec_nonfinite<BF16>(u32x4 x) { return dec_exponent_full<0x7f80u>(x); }
template <>
__device__ __forceinline__ bool dec_nonfinite<F16>(u32x4 x) { return dec_exponent_full<0x7c00u>(x); }

// Tiles of KT keys of a head: its cache's, then those of `fresh` new rows.
template <int KT>
__device__ __forceinline__ int dec_tiles(int n, int fresh) { return (n + KT - 1) / KT + (fresh + KT - 1) / KT; }
// A split's tiles: whole rounds of PER.
template <int PER>
__device__ __forceinline__ int dec_split(int tiles, int S) { return ((tiles + PER * S - 1) / (PER * S)) * PER; }

// A block's part of NB blocks that BH <= 128 heads share (NB >= 2 BH): tiles t0 .. t1 - 1 of a head of n rows, which has
// the blocks first .. first + count - 1. Every block takes `share` tiles (a multiple of per) of one head, the least
// that the blocks suffice for: long heads get many blocks.
struct DecPart {
  int bh, n, t0, t1, first, count;
};
template <int KT>
__device__ __forceinline__ bool dec_assign(DecI32In length, int BH, int C, int fresh, int NB, int per, DecPart& part) {
  const int lane = threadIdx.x & 63;       // a lane has heads `lane` and `lane + 64`
  int at[2], own[2], end[2];
  u32 tl[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) at[i] = length[min(lane + 64 * i, BH - 1)];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    at[i] = min(max(at[i], 0), C);
    tl[i] = lane + 64 * i < BH ? (u32)dec_tiles<KT>(at[i], fresh) : 0u;
  }
  u32 share = ((u32)__builtin_amdgcn_readlane(wave_inclusive_scan((int)(tl[0] + tl[1])), 63) + NB - 1) / NB;
  share = (share + per - 1) / per * per;
  while (true) {                            // (ends: total / share + BH blocks are enough)
#pragma unroll
    for (int i = 0; i < 2; ++i) own[i] = (int)((tl[i] + share - 1) / share);
    end[0] = wave_inclusive_scan(own[0]);
    end[1] = __builtin_amdgcn_readlane(end[0], 63) + wave_inclusive_scan(own[1]);
    if (__builtin_amdgcn_readlane(end[1], 63) <= NB) break;
    share += per * (1 + share / (16 * per));
  }
  const unsigned long long in0 = __ballot(end[0] > (int)blockIdx.x), in1 = __ballot(end[1] > (int)blockIdx.x);
  if (!in1) return false;
  const int from = __ffsll(in0 ? in0 : in1) - 1;
  part.bh = from + (in0 ? 0 : 64);
  part.n = __builtin_amdgcn_readlane(in0 ? at[0] : at[1], from);
  part.count = __builtin_amdgcn_readlane(in0 ? own[0] : own[1], from);
  part.first = __builtin_amdgcn_readlane(in0 ? end[0] : end[1], from) - part.count;
  part.t0 = ((int)blockIdx.x - part.first) * (int)share;
  part.t1 = min(dec_tiles<KT>(part.n, fresh), part.t0 + (int)share);
  return true;
}

// Zeros in place of the rows past the last (V: 0 * inf is not 0).
template <int DP, int NT, int NL>
__device__ __forceinline__ void dec_cut_rows(int kb, int rows, int tid, u32x4 (&x)[NL]) {
#pragma unroll
  for (int i = 0; i < NL; ++i)
    if (kb + (i * NT + tid) / (DP / 8) >= rows) x[i] = (u32x4){0u, 0u, 0u, 0u};
}

template <typename E>
__device__ __forceinline__ f32x4 dec_mfma16(u32x4 x, u32x4 y, f32x4 c);
template <>
__device__ __forceinline__ f32x4 dec_mfma16<BF16>(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 dec_mfma16<F16>(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// Maximum and sum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (the four that hold a query's keys).
__device__ __forceinline__ float dec_quad_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float dec_quad_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Block (split, KV head, batch row). S^T = K Q^T and O^T = V^T P^T with the 16 rows in the lanes' low four bits: 32 keys
// are two accumulators of S^T, whose registers (keys 4 (lane / 16) + i of each) are P^T's operand as
// they are; V^T's comes from transposing reads in that key order.
// Waves take keys for themselves, without a barrier, for the tile of 16 rows leaves the matrix pipe idle most of the time.
// What bounds it: HBM where the cache is long (the next 32 keys' K and V are on their way to registers while a wave
// works on these): 131072 rows of 8 heads, 128 channels, 110 us, 4.9 TB/s. Where it is short, the reading of its own code
// and the round trips to memory: 1024 rows 6.1 us.
template <typename E, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void decode_few_kernel(const DecArgs args) {
  constexpr int NC = DP / 32, NT16 = DP / 16, CPR = DP / 8, NL = DP / 16, TILE = 64 * DP, OST = DP + 4, RS = 16;
  constexpr int WLDS = 2 * TILE;         // a wave's LDS: a K and a V tile, then its output
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][WLDS];
  __shared__ float sm[3][4][RS];
  static_assert(WLDS >= RS * OST * 4 && WLDS >= (32 * RS + DP) * 4, "output, or probabilities and a value, in a wave's tiles");
  const DecArgs a = dec_hold(args);
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int hkv = (int)blockIdx.y, b = (int)blockIdx.z, bh = b * (int)gridDim.y + hkv, n, t0 = 0, t1 = 0;
  long long slot = (long long)bh * a.S + blockIdx.x;
  if (a.NB) {
    DecPart p;
    if (!dec_assign<32>(a.length, a.BH, a.C, a.T, a.NB, 4, p)) return;
    bh = p.bh, n = p.n, t0 = p.t0, t1 = p.t1, slot = blockIdx.x;
    b = bh / a.Hkv, hkv = bh - b * a.Hkv;
    if (t0 == 0 && threadIdx.x < 2) a.heads[2 * bh + threadIdx.x] = threadIdx.x ? p.count : p.first;
  } else {
    n = a.length[bh];
  }
  // this lane's query row (row 0 where there is none: its results go nowhere)
  const int r = l16 < a.R ? l16 : 0, g = a.T == 1 ? r : r / a.T, tq = r - g * a.T;
  u32x4 qf[NC];
  {
    const DecIn qp = a.q + b * a.qb + (long long)(hkv * (a.R / a.T) + g) * a.qh + tq * a.qn;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = *(const FE_GLOBAL u32x4*)(qp + (DP == a.D || 32 * c + 8 * lq < a.D ? 32 * c + 8 * lq : 0));
  }
  if (a.D != DP) {
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] &= 32 * c + 8 * lq < a.D ? ~0u : 0u;
  }
  const DecIn kc = a.kc + b * a.kcb + hkv * a.kch, vc = a.vc + b * a.vcb + hkv * a.vch;
  const DecIn kn = a.k + b * a.kb + hkv * a.kh, vn = a.v + b * a.vb + hkv * a.vh;
  n = __builtin_amdgcn_readfirstlane(min(max(n, 0), a.C));
  const int nc = (n + 31) / 32;
  if (!a.NB) {
    const int tiles = nc + (a.T + 31) / 32, share = dec_split<4>(tiles, a.S);
    t0 = (int)blockIdx.x * share, t1 = min(tiles, t0 + share);
    if (t0 >= t1) return;
  }

  unsigned char* kt = lds[wv];
  unsigned char* vt = lds[wv] + TILE;
  f32x4 o[NT16];
  float m = kDecNegInf, l = 0.f, lr = 0.f;   // l, lr: of the lane's keys
#pragma unroll
  for (int i = 0; i < NT16; ++i) o[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 kx[NL] = {}, vx[NL] = {};
  int t = -1, next = t0 + wv;
#pragma unroll 1
  while (true) {
    const bool tail = t >= nc;
    const int kb = (tail ? t - nc : t) * 32, rows = tail ? a.T : n;
    u32 odd = 0;                           // keys of new rows whose value has an infinity or a NaN
    if (t >= 0) {
      if (kb + 32 > rows) dec_cut_rows<DP, 64>(kb, rows, lane, vx);
      if (a.D != DP) {
        int D = a.D;
        asm volatile("" : "+s"(D));
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (8 * ((i * 64 + lane) % CPR) >= D) kx[i] = (u32x4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int e = i * 64 + lane;
        *(u32x4*)(kt + dec_k_at<DP>(e / CPR, e % CPR)) = kx[i];
        *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = vx[i];
      }
      if (tail) {
        u32 bad = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) bad |= dec_nonfinite<E>(vx[i]) ? 1u << ((i * 64 + lane) / CPR) : 0u;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) bad |= __shfl_xor(bad, d);
        odd = __builtin_amdgcn_readfirstlane(bad);
      }
    }
    if (next < t1) {
      const bool nt = next >= nc;
      const int nkb = (nt ? next - nc : next) * 32, last = (nt ? a.T : n) - 1;
      const DecIn kp = nt ? kn : kc, vp = nt ? vn : vc;
      const u32 ks = nt ? a.kn : a.kcn, vs = nt ? a.vn : a.vcn;
      int D = a.D;
      asm volatile("" : "+s"(D));          // compared here, not kept as masks over the loop
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int e = i * 64 + lane, ch = 8 * (e % CPR);
        const u32 row = (u32)min(nkb + e / CPR, last);
        const int cc = ch < D ? ch : 0;
        kx[i] = *(const FE_GLOBAL u32x4*)(kp + (unsigned long long)row * ks + cc);
        vx[i] = *(const FE_GLOBAL u32x4*)(vp + (unsigned long long)row * vs + cc);
      }
    }
    if (t >= 0) {
      // 0 * inf would reach the rows that do not see such a key, so its value is taken out of the product, and
      // added to the rows that do
      if (odd) {
        dec_wave_order();
        for (int e = lane; e < 32 * CPR; e += 64)
          if ((odd >> (e / CPR)) & 1u) *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = (u32x4){0u, 0u, 0u, 0u};
      }
      dec_wave_order();
      f32x4 x[2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const u32x4 kf = *(const u32x4*)(kt + dec_k_at<DP>(16 * s + l16, 4 * c + lq));
          x[s] = dec_mfma16<E>(kf, qf[c], c == 0 ? (f32x4){0.f, 0.f, 0.f, 0.f} : x[s]);
        }
      u32x4 pf;
      u32 vis = 0xffu;                      // bit 4 s + i: register i of x[s], key kb + 16 s + 4 lq + i, is visible
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i >> 2][i & 3] *= a.scale_log2;
      if (tail || kb + 32 > rows) {
        const FE_GLOBAL unsigned char* row = a.tree + b * a.tree_stride + tq * a.T;
        vis = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = kb + 16 * (i >> 2) + 4 * lq + (i & 3);
          bool see = key < rows;
          if (tail) see = see && (a.tree ? row[see ? key : 0] != 0 : key <= tq);
          vis |= (see ? 1u : 0u) << i;
          x[i >> 2][i & 3] = see ? x[i >> 2][i & 3] : kDecNegInf;
        }
      }
      float mn = kDecNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = fmaxf(mn, x[i >> 2][i & 3]);
      if (a.logits && l16 < a.R) {
        const DecF32 lp = a.logits + (((long long)bh * a.max_tiles + t) * a.R + l16) * 32 + 4 * lq;
        *(FE_GLOBAL f32x4*)lp = x[0];
        *(FE_GLOBAL f32x4*)(lp + 16) = x[1];
      }
      mn = fmaxf(m, dec_quad_max(mn));
      const float ref = mn == kDecNegInf ? 0.f : mn;
      const float alpha = fast_exp2(m - ref);
      m = mn;
      float ls = 0.f, lrs = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i >> 2][i & 3] = fast_exp2(x[i >> 2][i & 3] - ref);
        ls += x[i >> 2][i & 3];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pf[i] = E::pack2(x[i >> 1][2 * (i & 1)], x[i >> 1][2 * (i & 1) + 1]);
        lrs += E::to_f32((u16)pf[i]) + E::to_f32((u16)(pf[i] >> 16));
      }
      l = l * alpha + ls;
      lr = lr * alpha + lrs;
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int i = 0; i < NT16; ++i) o[i] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < NT16; ++i) {
        // channels 16 i + l16: keys 4 lq .. + 3, then 16 + 4 lq .. + 3
        const int row = 4 * lq + (l16 >> 2);
        unsigned char* p = vt + row * (DP * 2) + ((i >> 1) ^ dec_vswz<DP>(row)) * 64 + 32 * (i & 1) + 8 * (l16 & 3);
        const u32x2 ux = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)p));
        const u32x2 uy = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)(p + 16 * DP * 2)));
        o[i] = dec_mfma16<E>((u32x4){ux[0], ux[1], uy[0], uy[1]}, pf, o[i]);
      }
      if (odd) {
        dec_wave_order();
        float* sp = (float*)kt;             // [32 keys][RS rows] probabilities (-1: hidden)
        float* val = sp + 32 * RS;          // a value's channels
#pragma unroll
        for (int i = 0; i < 8; ++i) sp[(16 * (i >> 2) + 4 * lq + (i & 3)) * RS + l16] = (vis >> i) & 1u ? x[i >> 2][i & 3] : -1.f;
        for (u32 left = odd; left; left &= left - 1) {
          const int key = __ffs((int)left) - 1;
          for (int ch = lane; ch < DP; ch += 64) val[ch] = ch < a.D ? E::to_f32(vn[(unsigned long long)(kb + key) * a.vn + ch]) : 0.f;
          dec_wave_order();
          const float p = sp[key * RS + l16];
#pragma unroll
          for (int i = 0; i < NT16; ++i) {
            const f32x4 y = *(const f32x4*)(val + 16 * i + 4 * lq);
            if (p >= 0.f || p != p) o[i] += p * y;
          }
          dec_wave_order();
        }
      }
      dec_wave_order();                     // the next tile's stores follow this one's reads
    }
    if (next >= t1) break;
    t = next;
    next += 4;
  }

  // join the four waves (waves without a tile have a maximum of -inf and zeros)
  float* mine = (float*)lds[wv];
  l = dec_quad_sum(l);
  lr = dec_quad_sum(lr);
  if (lq == 0) {
    sm[0][wv][l16] = m;
    sm[1][wv][l16] = l;
    sm[2][wv][l16] = lr;
  }
#pragma unroll
  for (int i = 0; i < NT16; ++i) *(f32x4*)(mine + l16 * OST + 16 * i + 4 * lq) = o[i];
  __syncthreads();
#pragma unroll 1
  for (int e = threadIdx.x; e < a.R * (DP / 4); e += 256) {
    const int row = e / (DP / 4), ch = 4 * (e % (DP / 4));
    const float mx = fmaxf(fmaxf(sm[0][0][row], sm[0][1][row]), fmaxf(sm[0][2][row], sm[0][3][row]));
    const float ref = mx == kDecNegInf ? 0.f : mx;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    float lt = 0.f, lrt = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = fast_exp2(sm[0][i][row] - ref);
      s += w * *(const f32x4*)((float*)lds[i] + row * OST + ch);
      lt += w * sm[1][i][row];
      lrt += w * sm[2][i][row];
    }
    // partials are normalised by the sum of the rounded probabilities, and weighted by the exact one: so a row
    // that one key dominates returns that key's value whatever the split
    *(FE_GLOBAL f32x4*)(a.part_o + (slot * RS + row) * DP + ch) = s * (lrt == 0.f ? 0.f : __builtin_amdgcn_rcpf(lrt));
    if (ch == 0) {
      a.part_ml[slot * 2 * RS + row] = mx;
      a.part_ml[slot * 2 * RS + RS + row] = lt;
    }
  }
}

// Block (split, KV head, row block of a batch row). A wave holds 32 of its rows; the block's waves share tiles of 64 keys,
// whose loads are on the way to registers during the tile before. A row keeps its reference maximum until a tile's
// probabilities could overflow (E::kMaxTileSum), as in the prefill kernels, so most tiles spend nothing on maxima and
// rescaling. The two waves of a SIMD run half a tile apart: one multiplies a tile's probabilities by V right away, the
// other at the next tile, while the first is at its exponentials.
// What bounds it: the matrix pipe and the vector work beside it, 6.7 vector instructions to a product, an exponential a
// logit among them, which together fill 85% of a SIMD's time though they could overlap; LDS is busy 26% of it. Trees of
// 61 tokens of 7 heads over 4 KV heads' 32768 and 24576 rows, 128 channels: 74 us, 680 TFLOP/s (fp16); of 64 tokens of 4
// heads over 64 heads of 2304 to 4096 rows: 48 us, 570 TFLOP/s, 2.2 TB/s.
// One barrier a tile and the waves in step: 5% slower; four waves a block and two blocks a CU: 14% (tree of 64).
template <typename E, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP > 128 ? 1 : 2) void decode_wide_kernel(const DecArgs args) {
  constexpr int NDC = DP / 16, NDT = DP / 32, CPR = DP / 8, TILE = 128 * DP;   // bytes of 64 rows
  constexpr int NT = NW * 64, NL = (64 * CPR + NT - 1) / NT, OST = DP + 4;
  // eight waves: two on a SIMD. K of two tiles; V of three then: waves that run late read the tile before while the
  // next one comes in
  constexpr int VB = NW == 8 ? 3 : 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[(2 + VB) * TILE];
  __shared__ u32 s_odd[kDecMaxTokens / 64][2];   // keys of the tiles of new rows whose value has an infinity or a NaN
  __shared__ u32 s_tree[kDecMaxTokens][2];   // what each query token sees of a tile of new rows
  static_assert((2 + VB) * TILE >= NW * 16 * OST * 4, "16 rows of each wave's output");
  const DecArgs a = dec_hold(args);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool late = VB == 3 && wv >= 4;
  u32 ones2;
  asm volatile("s_mov_b32 %0, %1" : "=s"(ones2) : "i"(E::kOnes2));
  const int rb = (int)blockIdx.y;
  int bh = (int)blockIdx.x, n, t0 = 0, t1;
  if (a.NB) {
    DecPart p;
    if (!dec_assign<64>(a.length, a.BH, a.C, a.T, a.NB, 1, p)) return;
    bh = p.bh, n = p.n, t0 = p.t0, t1 = p.t1;
    if (t0 == 0 && rb == 0 && tid < 2) a.heads[2 * bh + tid] = tid ? p.count : p.first;
  } else {
    n = __builtin_amdgcn_readfirstlane(min(max(a.length[bh], 0), a.C));
    t1 = dec_tiles<64>(n, a.T);
    if (rb == 0 && tid < 2) a.heads[2 * bh + tid] = tid ? 1 : bh;
  }
  const int b = bh / a.Hkv, hkv = bh - b * a.Hkv, nc = (n + 63) / 64;
  {
    const int r = rb * a.RS + wv * 32 + l32;
    const bool live = wv * 32 < a.RS && rb * a.RS + wv * 32 < a.R;   // the wave has rows
    const bool rv = live && r < a.R;
    const int g = rv ? r / a.T : 0, tq = rv ? r - g * a.T : 0;
    const DecIn kc = a.kc + b * a.kcb + hkv * a.kch, vc = a.vc + b * a.vcb + hkv * a.vch;
    const DecIn kn = a.k + b * a.kb + hkv * a.kh, vn = a.v + b * a.vb + hkv * a.vh;
    u32x4 qf[NDC];
    {
      const DecIn qp = a.q + b * a.qb + (long long)(hkv * (a.R / a.T) + g) * a.qh + tq * a.qn;
      int D = a.D;
      asm volatile("" : "+s"(D));
#pragma unroll
      for (int c = 0; c < NDC; ++c) qf[c] = *(const FE_GLOBAL u32x4*)(qp + (16 * c + 8 * hh < D ? 16 * c + 8 * hh : 0));
    }
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = (f32x16){};
    float m = kDecNegInf, nm = 0.f, l = 0.f, lr = 0.f;   // lane-wise sums (half of a row's keys each)
    u32x4 kx[NL] = {}, vx[NL] = {};
    // a tile's rows on their way (past the last, the last), and into LDS
    auto load = [&](int t) __attribute__((always_inline)) {
      const bool nt = t >= nc;
      const int kb = (nt ? t - nc : t) * 64, last = (nt ? a.T : n) - 1;
      const DecIn kp = nt ? kn : kc, vp = nt ? vn : vc;
      const u32 ks = nt ? a.kn : a.kcn, vs = nt ? a.vn : a.vcn;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int e = i * NT + tid, ch = 8 * (e % CPR);
        const u32 row = (u32)min(kb + e / CPR, last);
        const int cc = ch < a.D ? ch : 0;
        kx[i] = *(const FE_GLOBAL u32x4*)(kp + (unsigned long long)row * ks + cc);
        vx[i] = *(const FE_GLOBAL u32x4*)(vp + (unsigned long long)row * vs + cc);
      }
    };
    auto kbuf = [&](int t) -> unsigned char* { return lds + (t & 1) * TILE; };
    auto vbuf = [&](int t) -> unsigned char* { return lds + (2 + t % VB) * TILE; };
    auto store = [&](int t) __attribute__((always_inline)) {
      unsigned char* kt = kbuf(t);
      unsigned char* vt = vbuf(t);
      const bool nt = t >= nc;
      const int kb = (nt ? t - nc : t) * 64, rows = nt ? a.T : n;
      dec_cut_rows<DP, NT>(kb, rows, tid, vx);   // (unconditionally, as below)
      if (a.D != DP) {
        int D = a.D;
        asm volatile("" : "+s"(D));
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (8 * ((i * NT + tid) % CPR) >= D) kx[i] = (u32x4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int e = i * NT + tid;
        if (64 * CPR % NT == 0 || e < 64 * CPR) {
          *(u32x4*)(kt + dec_k_at<DP>(e / CPR, e % CPR)) = kx[i];
          *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = vx[i];
        }
      }
      if (nt) {
        if (tid < 2) s_odd[t - nc][tid] = 0u;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int key = (i * NT + tid) / CPR;
          if (key < 64 && dec_nonfinite<E>(vx[i])) atomicOr(&s_odd[t - nc][key >> 5], 1u << (key & 31));
        }
      }
    };
    load(t0);
    // (unconditionally: fragments changed in a branch cost 250 spilled registers)
#pragma unroll
    for (int c = 0; c < NDC; ++c) {
      const u32 keep = rv && 16 * c + 8 * hh < a.D ? a.qand : 0u, flip = keep ? a.qxor : 0u;
      qf[c] = (qf[c] & keep) ^ flip;
    }
    store(t0);
    // 256 channels leave no registers for rows on their way: 256 rows of 8 heads over 8192 rows 114 us with them, 59 without
    constexpr bool AHEAD = DP <= 192;
    if (AHEAD && t0 + 1 < t1) load(t0 + 1);
    __syncthreads();
    // the next tile into LDS, the one behind it on its way
    auto advance = [&](int t) __attribute__((always_inline)) {
      if (!AHEAD && t + 1 < t1) load(t + 1);
      if (t + 1 < t1) store(t + 1);
      if (AHEAD && t + 2 < t1) load(t + 2);
      __syncthreads();
    };
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      {
        const bool tail = t >= nc;
        const int kb = (tail ? t - nc : t) * 64, rows = tail ? a.T : n;
        unsigned char* kt = kbuf(t);
        if (tail) {
          if (a.tree) {
            // the tile's columns of the mask, a query token a ballot
            // 16 on their way at once: a trip each had been most of a short call's time (854 rows of 44 heads over 143 rows,
            // 192 channels: 87 us)
            const FE_GLOBAL unsigned char* row = a.tree + b * a.tree_stride + min(kb + lane, a.T - 1);
#pragma unroll 1
            for (int u = wv; u < a.T; u += 16 * NW) {
              unsigned char see[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) see[i] = row[min(u + i * NW, a.T - 1) * a.T];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const unsigned long long sees = __ballot(see[i] != 0);
                if (lane < 2 && u + i * NW < a.T) s_tree[u + i * NW][lane] = (u32)(sees >> (32 * lane));
              }
            }
          }
          // 0 * inf would reach the rows that do not see such a key: its value is taken out of the product, and added
          // to the rows that do after the last tile
          const unsigned long long odd = ((unsigned long long)s_odd[t - nc][1] << 32) | s_odd[t - nc][0];
          if (odd)
            for (int e = tid; e < 64 * CPR; e += NT)
              if ((odd >> (e / CPR)) & 1u) *(u32x4*)(vbuf(t) + dec_v_at<DP>(e / CPR, e % CPR)) = (u32x4){0u, 0u, 0u, 0u};
          __syncthreads();
        }
        u32x4 pf[4] = {};                  // the tile's probabilities, as the product takes them
        if (live) {
          u32 vis[2] = {~0u, ~0u};         // bit 8 (i / 4) + i % 4 of word s: register i of x[s] is of a visible key
          const bool masked = tail || kb + 64 > rows;
          if (masked) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const int left = rows - kb - 32 * s, own = tq - kb - 32 * s + 1;
              u32 x = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u;
              if (tail) x &= a.tree ? s_tree[tq][s] : own >= 32 ? ~0u : own > 0 ? (1u << own) - 1u : 0u;
              vis[s] = x >> (4 * hh);
            }
          }
          f32x16 x[2];                     // logits, then probabilities
          auto logits = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
              for (int c = 0; c < NDC; ++c) {
                if (c % 4 == 0) __builtin_amdgcn_sched_barrier(0);   // four fragments in flight
                x[s] = c == 0 ? E::mfma(dec_kfrag<DP>(kt, 32 * s, 0), qf[0], (f32x16){}) : E::mfma(dec_kfrag<DP>(kt, 32 * s, c), qf[c], x[s]);
              }
            }
            if (masked) {
#pragma unroll
              for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const u32 on = (u32)((int)(vis[s] << (31 - 8 * (i >> 2) - (i & 3))) >> 31);
                  x[s][i] = __uint_as_float((__float_as_uint(x[s][i]) & on) | (0xff800000u & ~on));
                }
            }
          };
          float ls;
          auto exponentials = [&]() __attribute__((always_inline)) {
            ls = 0.f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                x[s][i] = fast_exp2(x[s][i] * a.scale_log2 + nm);
                ls += x[s][i];
              }
          };
          logits();
          exponentials();
          const bool over = !(ls <= E::kMaxTileSum) || m == kDecNegInf;
          if (__ballot(over)) {
            // a new reference for rows without one, and for those whose probabilities grew too large
            logits();
            float mx = kDecNegInf;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[s][i]);
            mx = half_swap_max(mx) * a.scale_log2;
            const bool take = half_swap_max(over ? 1.f : 0.f) > 0.f && mx > m;
            const float alpha = !take ? 1.f : m == kDecNegInf ? 0.f : fast_exp2(m - mx);
            m = take ? mx : m;
            nm = take ? -mx : nm;
            l *= alpha;
            lr *= alpha;
            // in place: left to the compiler, every tile copies the accumulators for the rare one that scales them
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
              for (int i = 0; i < 16; ++i) asm volatile("v_mul_f32 %0, %1, %0" : "+v"(o[dt][i]) : "v"(alpha));
            exponentials();
          }
          l += ls;
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              pf[c4][i] = E::pack2(x[c4 >> 1][8 * (c4 & 1) + 2 * i], x[c4 >> 1][8 * (c4 & 1) + 2 * i + 1]);
              lr = E::sum2(pf[c4][i], ones2, lr);
            }
        }
        // every wave meets the same barriers, the late ones' before the product
        if (late) advance(t);
        if (live) {
          unsigned char* vt = vbuf(t);
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] = E::mfma(dec_vfrag<DP>(vt, 16 * c4, dt), pf[c4], o[dt]);
        }
        if (!late) advance(t);
      }
    }
    if (live) {
#pragma unroll 1
      for (int t = max(t0, nc); t < t1; ++t) {
        const u32 lo = __builtin_amdgcn_readfirstlane(s_odd[t - nc][0]), hi = __builtin_amdgcn_readfirstlane(s_odd[t - nc][1]);
#pragma unroll 1
        for (unsigned long long odd = ((unsigned long long)hi << 32) | lo; odd; odd &= odd - 1) {
          const int u = (t - nc) * 64 + __ffsll(odd) - 1;
          const DecIn kp = kn + (unsigned long long)u * a.kn, vp = vn + (unsigned long long)u * a.vn;
          int D = a.D;
          asm volatile("" : "+s"(D));    // or its comparisons are kept over the loop
          float x = 0.f;
#pragma unroll
          for (int c = 0; c < NDC; ++c) {
            const int ch = 16 * c + 8 * hh;
            const u32x4 kk = ch < D ? *(const FE_GLOBAL u32x4*)(kp + ch) : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              x = __builtin_fmaf(E::to_f32((u16)kk[w]), E::to_f32((u16)qf[c][w]), x);
              x = __builtin_fmaf(E::to_f32((u16)(kk[w] >> 16)), E::to_f32((u16)(qf[c][w] >> 16)), x);
            }
          }
          const float pr = fast_exp2(half_swap_sum(x) * a.scale_log2 + nm);
          const bool sees = rv && (a.tree ? a.tree[b * a.tree_stride + tq * a.T + u] != 0 : u <= tq);
#pragma unroll
          for (int i = 0; i < 4 * NDT; ++i) {
            const int ch = 8 * i + 4 * hh;
            const u32x2 y = ch < D ? *(const FE_GLOBAL u32x2*)(vp + ch) : (u32x2){0u, 0u};
#pragma unroll
            for (int w = 0; w < 4; ++w)
              o[i >> 2][4 * (i & 3) + w] += sees ? pr * E::to_f32((u16)(y[w >> 1] >> (16 * (w & 1)))) : 0.f;
          }
        }
      }
    }
    __syncthreads();                       // LDS is the outputs' from here on
    l = half_swap_sum(l);
    lr = half_swap_sum(lr);
    const long long slot = (long long)blockIdx.x * a.RB + rb;
    if (live) {
      const float inv = lr == 0.f ? 0.f : 1.f / lr;
      if (rv && hh == 0) {
        a.part_ml[slot * 2 * a.RS + wv * 32 + l32] = m;
        a.part_ml[slot * 2 * a.RS + a.RS + wv * 32 + l32] = l;
      }
      // 16 rows at a time through LDS, so that rows are stored whole
      float* mine = (float*)lds + wv * 16 * OST;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        if ((l32 >> 4) == half) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *(f32x4*)(mine + (l32 & 15) * OST + 32 * dt + 8 * i + 4 * hh) =
                  (f32x4){o[dt][4 * i] * inv, o[dt][4 * i + 1] * inv, o[dt][4 * i + 2] * inv, o[dt][4 * i + 3] * inv};
        }
        dec_wave_order();
        const int row0 = wv * 32 + 16 * half, rows = min(16, a.R - rb * a.RS - row0);
#pragma unroll 4
        for (int e = lane; e < rows * (DP / 4); e += 64)
          *(FE_GLOBAL f32x4*)(a.part_o + (slot * a.RS + row0) * DP + 4 * e) = *(const f32x4*)(mine + e / (DP / 4) * OST + 4 * (e % (DP / 4)));
        dec_wave_order();
      }
    }
  }
}

// 32 rows a block, keys to its waves 32 at a time, everything read element by element. What bounds it: the instructions
// that put elements together.
template <typename E, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void decode_elements_kernel(const DecArgs a) {
  constexpr int NDC = DP / 16, NDT = DP / 32, CPR = DP / 8, TILE = 64 * DP;   // bytes of 32 rows
  constexpr int OST = 33;                // floats of a channel's 32 rows in LDS, and one against bank conflicts
  constexpr int WLDS = DP * OST * 4;     // a wave's LDS: a K and a V tile, then its output
  static_assert(WLDS >= 2 * TILE, "tiles");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][WLDS];
  __shared__ float sm[4][3][32];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned char* kt = lds[wv];
  unsigned char* vt = lds[wv] + TILE;

  const int hkv = (int)blockIdx.y, z = (int)blockIdx.z, b = z / a.RB, rb = z - b * a.RB, bh = b * (int)gridDim.y + hkv;
  const int n = __builtin_amdgcn_readfirstlane(min(max(a.length[bh], 0), a.C));
  const int nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.T), share = dec_split<4>(tiles, a.S);
  const int t0 = (int)blockIdx.x * share, t1 = min(tiles, t0 + share);
  if (t0 >= t1) return;
  {
    const int r = rb * 32 + l32;         // this lane's query row
    const bool rv = r < a.R;
    const int g = rv ? r / a.T : 0, tq = rv ? r - g * a.T : 0;
    const DecIn kc = a.kc + b * a.kcb + hkv * a.kch, vc = a.vc + b * a.vcb + hkv * a.vch;
    const DecIn kn = a.k + b * a.kb + hkv * a.kh, vn = a.v + b * a.vb + hkv * a.vh;
    u32x4 qf[NDC];
    {
      const DecIn qp = a.q + b * a.qb + (long long)(hkv * (a.R / a.T) + g) * a.qh + tq * a.qn;   // a real row in any case
#pragma unroll
      for (int c = 0; c < NDC; ++c) {
        qf[c] = (dec_load8(qp, a.qc, 2 * c + hh, a.D) & a.qand) ^ a.qxor;
        __builtin_amdgcn_sched_barrier(0);   // one chunk's addresses at a time
      }
    }
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = (f32x16){};
    float m = kDecNegInf, l = 0.f, lr = 0.f;   // sums of the probabilities, and of these as rounded for the product

    for (int t = t0 + wv; t < t1; t += 4) {
      const bool tail = t >= nc;
      const int kb = (tail ? t - nc : t) * 32, rows = tail ? a.T : n;
      const DecIn kp = tail ? kn : kc, vp = tail ? vn : vc;
      const long long krs = tail ? a.kn64 : a.kcn64, vrs = tail ? a.vn64 : a.vcn64, kcs = tail ? a.kd : a.kcd, vcs = tail ? a.vd : a.vcd;
      // keys of the tail whose value has an infinity or a NaN: 0 * inf would reach the rows that do not see
      // them, so their values are taken out of the product and added to the rows that do
      u32 odd = 0;
      {
#pragma unroll 1
        for (int i = 0; i < NDC; ++i) {
          const int e = i * 64 + lane, row = kb + e / CPR, ch = e % CPR;
          const u32x4 x = row < rows ? dec_load8(kp + row * krs, kcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
          *(u32x4*)(kt + dec_k_at<DP>(e / CPR, ch)) = x;
          __builtin_amdgcn_sched_barrier(0);
          const u32x4 y = row < rows ? dec_load8(vp + row * vrs, vcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
          *(u32x4*)(vt + dec_v_at<DP>(e / CPR, ch)) = y;
          if (tail)
            for (unsigned long long bl = __ballot(dec_nonfinite<E>(y)); bl; bl &= bl - 1) odd |= 1u << ((i * 64 + __ffsll(bl) - 1) / CPR);
        }
      }
      if (odd) {
        dec_wave_order();
        for (int e = lane; e < 32 * CPR; e += 64)
          if ((odd >> (e / CPR)) & 1u) *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = (u32x4){0u, 0u, 0u, 0u};
      }
      dec_wave_order();
      // S^T: lanes hold queries; register i holds key kb + 8 (i / 4) + 4 hh + i % 4
      f32x16 x;
#pragma unroll
      for (int c = 0; c < NDC; ++c) x = c == 0 ? E::mfma(dec_kfrag<DP>(kt, 0, 0), qf[0], (f32x16){}) : E::mfma(dec_kfrag<DP>(kt, 0, c), qf[c], x);
      u32 vis = ~0u;
      if (tail || kb + 32 > rows) {
        vis = 0;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const int key = kb + 8 * (i >> 2) + 4 * hh + (i & 3);
          bool see = key < rows;
          if (tail) see = see && (a.tree ? a.tree[b * a.tree_stride + tq * a.T + (see ? key : 0)] != 0 : key <= tq);
          vis |= (see ? 1u : 0u) << i;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = (vis >> i) & 1u ? x[i] : kDecNegInf;
      }
      float mn = kDecNegInf;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] *= a.scale_log2;
        mn = fmaxf(mn, x[i]);
      }
      if (a.logits && rv) {
        const DecF32 lp = a.logits + (((long long)bh * a.max_tiles + t) * a.R + r) * 32 + 4 * hh;
#pragma unroll
        for (int i = 0; i < 4; ++i) *(FE_GLOBAL f32x4*)(lp + 8 * i) = (f32x4){x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
      }
      mn = fmaxf(m, half_swap_max(mn));
      const float ref = mn == kDecNegInf ? 0.f : mn;
      const float alpha = fast_exp2(m - ref);
      m = mn;
      float ls = 0.f, lrs = 0.f;
      u32 pw[8];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = fast_exp2(x[i] - ref);
        ls += x[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pw[i] = E::pack2(x[2 * i], x[2 * i + 1]);
        lrs += E::to_f32((u16)pw[i]) + E::to_f32((u16)(pw[i] >> 16));
      }
      l = l * alpha + half_swap_sum(ls);
      lr = lr * alpha + half_swap_sum(lrs);
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
      }
#pragma unroll
      for (int c4 = 0; c4 < 2; ++c4) {
        const u32x4 pf = {pw[4 * c4], pw[4 * c4 + 1], pw[4 * c4 + 2], pw[4 * c4 + 3]};
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = E::mfma(dec_vfrag<DP>(vt, 16 * c4, dt), pf, o[dt]);
      }
      if (odd) {
        dec_wave_order();
        float* sp = (float*)kt;             // [32 keys][32 rows] probabilities (-1: hidden); K and V are done with
        float* row = sp + 1024;             // a value's channels
#pragma unroll
        for (int i = 0; i < 16; ++i) sp[(8 * (i >> 2) + 4 * hh + (i & 3)) * 32 + l32] = (vis >> i) & 1u ? x[i] : -1.f;
        for (u32 left = odd; left; left &= left - 1) {
          const int key = __ffs((int)left) - 1;
          for (int ch = lane; ch < DP; ch += 64) row[ch] = ch < a.D ? E::to_f32(vp[(kb + key) * vrs + ch * vcs]) : 0.f;
          dec_wave_order();
          const float p = sp[key * 32 + l32];
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float y = row[32 * dt + 8 * (i >> 2) + 4 * hh + (i & 3)];
              if (p >= 0.f) o[dt][i] += p * y;
            }
          dec_wave_order();
        }
      }
      dec_wave_order();                     // the next tile's stores follow this one's reads
    }

    // join the four waves
    if (hh == 0) {
      sm[wv][0][l32] = m;
      sm[wv][1][l32] = l;
      sm[wv][2][l32] = lr;
    }
    float* mine = (float*)lds[wv];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(32 * dt + 8 * (i >> 2) + 4 * hh + (i & 3)) * OST + l32] = o[dt][i];
    __syncthreads();
    const long long slot = ((long long)bh * a.RB + rb) * a.S + blockIdx.x;
    const int rows = min(32, a.R - rb * 32);
    for (int e = threadIdx.x; e < rows * DP; e += 256) {
      const int row = e / DP, ch = e % DP;
      float mx = fmaxf(fmaxf(sm[0][0][row], sm[1][0][row]), fmaxf(sm[2][0][row], sm[3][0][row]));
      const float ref = mx == kDecNegInf ? 0.f : mx;
      float s = 0.f, lt = 0.f, lrt = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = fast_exp2(sm[i][0][row] - ref);
        s += w * ((float*)lds[i])[ch * OST + row];
        lt += w * sm[i][1][row];
        lrt += w * sm[i][2][row];
      }
      // partials are normalised by the sum of the rounded probabilities, and weighted by the exact one: so a row
      // that one key dominates returns that key's value whatever the split
      a.part_o[(slot * 32 + row) * DP + ch] = lrt == 0.f ? 0.f : s * (1.f / lrt);
      if (ch == 0) {
        a.part_ml[slot * 64 + row] = mx;
        a.part_ml[slot * 64 + 32 + row] = lt;
      }
    }
  }
}

// Joins the splits. Blocks below out_blocks of a head: output rows, DP / 4 threads on a slot's values, merging slots as
// they are read (maximum, sum, values); where a row has many slots all of a block's groups of threads are on one row.
// The others, where there are logits: the head's importance, a tile of 32 keys to 32 lanes.
// What bounds it: two trips to memory and the reading of its code, 4.7 to 9 us; on long caches the logits' and weights'
// bytes: 8 heads of 131072 rows 13.3 us, 2.2 TB/s.
template <typename E, int DP>
__global__ __launch_bounds__(256) void decode_join_kernel(const DecJoinArgs args) {
  constexpr int LPR = DP / 4, NG = 256 / LPR, PF = 4;   // threads on a slot, groups of them; loads in flight
  __shared__ float sm[16][16], sl[16][16], bias[16];
  __shared__ f32x4 so[NG * LPR];
  const DecJoinArgs a = dec_hold(args);
  const int tid = threadIdx.x, hkv = (int)blockIdx.y, b = (int)blockIdx.z, bh = b * (int)gridDim.y + hkv;
  const int n = __builtin_amdgcn_readfirstlane(min(max(a.length[bh], 0), a.C));
  const int RS = a.RS;
  if ((int)blockIdx.x < a.out_blocks) {
    const int grp = tid / LPR, c4 = tid - grp * LPR;
    const int row = (int)blockIdx.x * a.rows + (a.rows > 1 ? grp : 0), step = a.rows > 1 ? 1 : NG;
    const bool rv = grp < NG && row < a.R;
    const int rb = a.RB == 1 ? 0 : row / RS;
    long long first = ((long long)bh * a.RB + rb) * a.S, pitch = RS;   // the row's slots: the first, values between them
    int count;
    if (a.heads) {
      first = (long long)a.heads[2 * bh] * a.RB + rb;
      count = a.heads[2 * bh + 1];
      pitch = (long long)RS * a.RB;
    } else {
      const int all = dec_tiles<32>(n, a.T), share = dec_split<4>(all, a.S);
      count = (all + share - 1) / share;
    }
    const DecF32In ml = a.part_ml + first * 2 * RS + (row - rb * RS);
    const DecF32In po = a.part_o + (first * RS + (row - rb * RS)) * DP + 4 * c4;
    float m = kDecNegInf, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s0 = a.rows > 1 ? 0 : grp; s0 < count && rv; s0 += PF * step) {
      float ms[PF], ls[PF];
      f32x4 x[PF];
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const int s = min(s0 + i * step, count - 1);
        ms[i] = ml[s * 2 * pitch];
        ls[i] = ml[s * 2 * pitch + RS];
        x[i] = *(const FE_GLOBAL f32x4*)(po + s * pitch * DP);
      }
#pragma unroll
      for (int i = 0; i < PF; ++i)
        if (i && s0 + i * step >= count) ms[i] = kDecNegInf, ls[i] = 0.f, x[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
      float mn = m;
#pragma unroll
      for (int i = 0; i < PF; ++i) mn = fmaxf(mn, ms[i]);
      const float ref = mn == kDecNegInf ? 0.f : mn, keep = fast_exp2(m - ref);
      l *= keep;
      acc *= keep;
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        // a split that this row sees nothing of has a weight of 0 and values of 0
        const float w = ls[i] * fast_exp2(ms[i] - ref);
        l += w;
        acc += w * x[i];
      }
      m = mn;
    }
    if (a.rows == 1) {
      if (grp < NG) {
        so[tid] = acc;
        if (c4 == 0) sm[0][grp] = m, sl[0][grp] = l;
      }
      __syncthreads();
      if (grp) return;
      float mx = m;
#pragma unroll
      for (int i = 1; i < NG; ++i) mx = fmaxf(mx, sm[0][i]);
      const float ref = mx == kDecNegInf ? 0.f : mx, keep = fast_exp2(m - ref);
      l *= keep;
      acc *= keep;
      m = mx;
#pragma unroll
      for (int i = 1; i < NG; ++i) {
        const float w = fast_exp2(sm[0][i] - ref);
        l += w * sl[0][i];
        acc += w * so[i * LPR + c4];
      }
    }
    if (!rv) return;
    acc *= l == 0.f ? 0.f : 1.f / l;
    const long long at = (long long)bh * a.R + row;       // [B, Hkv, G, T]
    const u32 w0 = E::pack2(acc[0], acc[1]), w1 = E::pack2(acc[2], acc[3]);
    FE_GLOBAL u16* op = a.out + at * a.D + 4 * c4;
    if (a.D % 4 == 0) {
      if (4 * c4 < a.D) *(FE_GLOBAL u32x2*)op = (u32x2){w0, w1};
    } else {
      const u16 h[4] = {(u16)w0, (u16)(w0 >> 16), (u16)w1, (u16)(w1 >> 16)};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * c4 + i < a.D) op[i] = h[i];
    }
    if (c4 == 0) a.lse[at] = l == 0.f ? kDecNegInf : (m + fast_log2(l)) * kLn2;
    return;
  }

  // a head's R <= kDecLogitRows rows, one row block; tiles of 32 keys
  const int nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.T), share = dec_split<4>(tiles, a.S);
  const int count = a.heads ? a.heads[2 * bh + 1] : (tiles + share - 1) / share;
  const long long first = a.heads ? a.heads[2 * bh] : (long long)bh * a.S;
  const int part = (int)blockIdx.x - a.out_blocks, step = 8 * ((int)gridDim.x - a.out_blocks), l32 = tid & 31;
  int t = part * 8 + (tid >> 5);
  if (part * 8 >= tiles) return;
  float x[PF], old = 0.f, w = 1.f;          // a tile's first rows of logits; its keys' importance and norms
  {
    const int row = tid & 15, grp = tid >> 4;
    const DecF32In ml = a.part_ml + first * 2 * RS + row;
    float m = kDecNegInf, l = 0.f;
    if (row < a.R) {
#pragma unroll 1
      for (int s = grp; s < count; s += 16) {
        const float ms = ml[(long long)s * 2 * RS], ls = ml[(long long)s * 2 * RS + RS];
        const float mn = fmaxf(m, ms), ref = mn == kDecNegInf ? 0.f : mn;
        l = l * fast_exp2(m - ref) + ls * fast_exp2(ms - ref);
        m = mn;
      }
    }
    sm[grp][row] = m;
    sl[grp][row] = l;
    __syncthreads();
    if (tid < 16) {
#pragma unroll 4
      for (int i = 1; i < 16; ++i) m = fmaxf(m, sm[i][row]);
      const float ref = m == kDecNegInf ? 0.f : m;
      l = 0.f;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) l += sl[i][row] * fast_exp2(sm[i][row] - ref);
      // log2 of l and of w = 2^(-decay (T - 1 - t)); rows that see nothing, or are none, give no weight
      bias[row] = l == 0.f || row >= a.R ? -kDecNegInf : ref + fast_log2(l) + a.decay_log2 * (float)(a.T - 1 - row % a.T);
    }
    __syncthreads();
  }
  const float keep = fast_exp2(-a.decay_log2 * (float)a.T);
#pragma unroll 1
  for (; t < tiles; t += step) {
    const DecF32In lp = a.logits + ((long long)bh * a.max_tiles + t) * a.R * 32 + l32;
    const int key = t * 32 + l32;
#pragma unroll
    for (int i = 0; i < PF; ++i) x[i] = lp[min(i, a.R - 1) * 32];
    if (key < n) {
      old = a.imp[bh * a.imp_stride + key];
      if (a.norm) w = a.norm[bh * a.norm_stride + key];
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PF; ++i) sum += fast_exp2(x[i] - bias[i]);
#pragma unroll 1
    for (int r0 = PF; r0 < a.R; r0 += PF) {
#pragma unroll
      for (int i = 0; i < PF; ++i) x[i] = lp[min(r0 + i, a.R - 1) * 32];
#pragma unroll
      for (int i = 0; i < PF; ++i) sum += fast_exp2(x[i] - bias[r0 + i]);
    }
    if (t < nc) {
      if (key < n) a.imp_out[bh * a.impo_stride + key] = old * keep + w * sum;
    } else if (key - nc * 32 < a.T) {
      const int u = key - nc * 32;
      float nu = 1.f;
      if (a.norm) {
        const DecIn vp = a.v + b * a.vb + hkv * a.vh + u * a.vn;
        nu = 0.f;
#pragma unroll 4
        for (int d = 0; d < a.D; ++d) nu += fabsf(E::to_f32(vp[d * a.vd]));
      }
      a.new_imp[(long long)bh * a.T + u] = nu * sum;
    }
  }
}

// Blocks as decode_few_kernel's. Rows r = g * A_b + i of the path, 64 to a wave, with their Q in registers as four tiles of
// 16; a wave takes 32 keys at a time, straight into the products' operands (a lane's 16 bytes of a key lie beside its
// neighbours' of the same key, 64 bytes in all), the next 32 on the way. Up to 64 rows, the block's waves take different
// keys; more, the same keys for 64 rows each, summed in LDS (132 rows of 2 heads and 3 batch rows over 5000 keys: 16.4 us
// with one wave for all of a key's rows, 10.4 so). More than 256 rows take K again, adding to what the rows before left.
// What bounds it: reading K, 24 rows of 4 heads and 8 batch rows of up to 32768 keys 54 us, 4.1 TB/s; on short caches the
// trips to memory one after the other (path, its rows, lse): 1024 keys 6.4 us.
template <typename E, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void decode_replay_kernel(const DecReplayArgs args) {
  constexpr int NC = DP / 32, RT = 4, CH = 16 * RT;
  __shared__ __attribute__((aligned(16))) float lse[4 * CH], weight[4 * CH];   // a row's, and log2 of w
  __shared__ int place[4 * CH], node[4 * CH];   // a row's index on the path, and its token
  __shared__ float s_sum[2][4][32];        // a tile's sums of the waves' rows
  const DecReplayArgs a = dec_hold(args);
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  int hkv = (int)blockIdx.y, b = (int)blockIdx.z, bh = b * (int)gridDim.y + hkv, n, t0 = 0, t1 = 0;
  if (a.NB) {
    DecPart p;
    if (!dec_assign<32>(a.length, a.BH, a.C, a.A, a.NB, a.G * a.A > CH ? 1 : 4, p)) return;
    bh = p.bh, n = p.n, t0 = p.t0, t1 = p.t1;
    b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  } else {
    n = a.length[bh];
  }
  const DecI32In path = a.path ? a.path + (long long)b * a.A : a.path;
  int na = a.A;
  if (path) {
    na = 0;
    for (int i0 = 0; i0 < a.A; i0 += 64) {
      const int x = path[min(i0 + lane, a.A - 1)];
      const unsigned long long ok = __ballot(i0 + lane < a.A && x >= 0 && x < a.T);
      const int run = ok == ~0ull ? 64 : __ffsll(~ok) - 1;
      na += run;
      if (run < 64) break;
    }
  }
  n = __builtin_amdgcn_readfirstlane(min(max(n, 0), a.C));
  const int nc = (n + 31) / 32;
  if (!a.NB) {
    const int tiles = nc + (a.A + 31) / 32, share = a.G * a.A > CH ? dec_split<1>(tiles, a.S) : dec_split<4>(tiles, a.S);
    t0 = (int)blockIdx.x * share, t1 = min(tiles, t0 + share);
    if (t0 >= t1) return;
  }
  const int rend = a.G * na, ws = rend > CH ? 4 : 1, rw = ws == 4 ? wv * CH : 0;   // the wave's rows in lse, weight, place, node
  const DecIn kc = a.kc + b * a.kcb + hkv * a.kch, kn = a.k + b * a.kb + hkv * a.kh;
  const float keep = fast_exp2(-a.decay_log2 * (float)na);

#pragma unroll 1
  for (int r0 = 0; r0 == 0 || r0 < rend; r0 += CH * ws) {
    __syncthreads();                        // the rows before are done with
    if (tid < CH * ws) {
      const int r = r0 + tid;
      float z = -kDecNegInf;                // no row: no weight
      int at = 0, nd = 0;
      if (r < rend) {
        const int g = r / na;
        at = r - g * na;
        nd = path ? path[at] : at;
        z = a.lse[((long long)bh * a.G + g) * a.T + nd];
        z = z == kDecNegInf ? -kDecNegInf : z;   // nothing visible: no weight
        nd |= g << 16;
      }
      lse[tid] = z;
      weight[tid] = a.decay_log2 * (float)(at + 1 - na);
      place[tid] = at;
      node[tid] = nd;
    }
    __syncthreads();
    u32x4 qf[RT][NC];
    f32x4 zs[RT], lw[RT];
    const int mine = rend - r0 - rw;        // rows from the wave's first on
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (16 * rt < mine) {
        const int nd = node[rw + 16 * rt + l16];   // a real row in any case
        const DecIn qp = a.q + b * a.qb + (long long)(hkv * a.G + (nd >> 16)) * a.qh + (nd & 0xffff) * a.qn;
#pragma unroll
        for (int c = 0; c < NC; ++c) qf[rt][c] = *(const FE_GLOBAL u32x4*)(qp + (DP == a.D || 32 * c + 8 * lq < a.D ? 32 * c + 8 * lq : 0));
        zs[rt] = *(const f32x4*)(lse + rw + 16 * rt + 4 * lq);
        lw[rt] = *(const f32x4*)(weight + rw + 16 * rt + 4 * lq);
      }
    }
    if (a.D != DP) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int c = 0; c < NC; ++c) qf[rt][c] &= 32 * c + 8 * lq < a.D ? ~0u : 0u;
    }
    u32x4 kx[2][NC];
    float ox = 0.f, wx = 1.f, old = 0.f, w = 1.f;   // importance and norm of key kb + lane (lanes below 32)
    int t = -1, next = ws == 4 ? t0 : t0 + wv;
#pragma unroll 1
    while (true) {
      u32x4 kf[2][NC];
      if (t >= 0) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int c = 0; c < NC; ++c) kf[s][c] = kx[s][c];
        if (a.D != DP) {
          int D = a.D;
          asm volatile("" : "+s"(D));
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < NC; ++c)
              if (32 * c + 8 * lq >= D) kf[s][c] = (u32x4){0u, 0u, 0u, 0u};
        }
        old = ox;
        w = wx;
      }
      if (next < t1) {
        const bool nt = next >= nc;
        const int kb = (nt ? next - nc : next) * 32;
        int D = a.D;
        asm volatile("" : "+s"(D));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32 row = (u32)min(kb + 16 * s + l16, nt ? max(na, 1) - 1 : n - 1);
          if (nt && path) row = (u32)min(max(path[row], 0), a.T - 1);   // new rows in the path's order
          const DecIn kp = (nt ? kn : kc) + (unsigned long long)row * (nt ? a.kn : a.kcn);
#pragma unroll
          for (int c = 0; c < NC; ++c) kx[s][c] = *(const FE_GLOBAL u32x4*)(kp + (32 * c + 8 * lq < D ? 32 * c + 8 * lq : 0));
        }
        if (!nt && lane < 32) {
          const int key = min(kb + lane, n - 1);
          ox = r0 ? a.imp_out[bh * a.impo_stride + key] : a.imp[bh * a.imp_stride + key];
          if (a.norm) wx = a.norm[bh * a.norm_stride + key];
        }
      }
      if (t >= 0) {
        const bool tail = t >= nc;
        const int kb = (tail ? t - nc : t) * 32;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (16 * rt < mine) {
            // lanes hold keys kb + 16 s + l16; register i holds row 16 rt + 4 lq + i
            f32x4 x[2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int c = 0; c < NC; ++c) x[s] = dec_mfma16<E>(qf[rt][c], kf[s][c], c == 0 ? (f32x4){0.f, 0.f, 0.f, 0.f} : x[s]);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i) x[s][i] = fast_exp2(__builtin_fmaf(__builtin_fmaf(x[s][i], a.scale, -zs[rt][i]), 1.f / kLn2, lw[rt][i]));
            if (tail || 16 * (rt + 1) > mine) {
              int left = mine;
              asm volatile("" : "+s"(left));   // compared here, not kept as masks across the loop
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int rr = 16 * rt + 4 * lq + i, at = place[rw + rr];
#pragma unroll
                for (int s = 0; s < 2; ++s)     // no row, whatever the key; row `at` of the path sees new row u <= at
                  if (rr >= left || (tail && at < kb + 16 * s + l16)) x[s][i] = 0.f;
              }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) sum[s] += (x[s][0] + x[s][1]) + (x[s][2] + x[s][3]);
          }
        }
        const float s0 = dec_quad_sum(sum[0]), s1 = dec_quad_sum(sum[1]);
        float total = lq == 0 ? s0 : s1;
        const int key = kb + lane;
        if (ws == 4) {
          if (lane < 32) s_sum[t & 1][wv][lane] = total;
          __syncthreads();
          const float(&part)[4][32] = s_sum[t & 1];
          total = (part[0][lane & 31] + part[1][lane & 31]) + (part[2][lane & 31] + part[3][lane & 31]);
        }
        if (ws == 4 && wv) {
          // the first wave's to write
        } else if (!tail) {
          if (lane < 32 && key < n) a.imp_out[bh * a.impo_stride + key] = old * (r0 ? 1.f : keep) + w * total;
        } else if (lane < 32 && key < a.A) {
          float nu = 1.f;
          if (a.norm && key < na) {
            const FE_GLOBAL u32x4* vp =
                (const FE_GLOBAL u32x4*)(a.v + b * a.vb + hkv * a.vh + (unsigned long long)(u32)(path ? path[key] : key) * a.vn);
            nu = 0.f;
            for (int d = 0; d < a.D / 8; ++d) {
              const u32x4 y = vp[d];
#pragma unroll
              for (int i = 0; i < 4; ++i) nu += fabsf(E::to_f32((u16)y[i])) + fabsf(E::to_f32((u16)(y[i] >> 16)));
            }
          }
          const DecF32 to = a.new_imp + (long long)bh * a.A + key;
          *to = (r0 ? *to : 0.f) + (key < na ? nu * total : 0.f);
        }
      }
      if (next >= t1) break;
      t = next;
      next += ws == 4 ? 1 : 4;
    }
  }
}

// Rows whose Q is in LDS at a time.
template <int DP>
constexpr int dec_replay_rows() { return DP > 128 ? 32 : 64; }

// Leading nodes of batch row b's path that name one of the T tokens.
__device__ __forceinline__ int dec_path_len(const DecReplayArgs& a, int b) {
  if (!a.path) return a.A;
  int len = 0;
  for (int i0 = 0; i0 < a.A; i0 += 64) {
    const int i = i0 + (int)(threadIdx.x & 63);
    const int node = i < a.A ? a.path[(long long)b * a.A + i] : -1;
    const unsigned long long ok = __ballot(node >= 0 && node < a.T);
    const int run = ok == ~0ull ? 64 : __ffsll(~ok) - 1;
    len += run;
    if (run < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(len);
}

// Any layout, element by element: a wave takes 32 keys at a time through its own LDS into registers, against the rows'
// Q in LDS. More rows than that has room for take K again, adding to what the rows before left.
template <typename E, int DP>
__global__ __launch_bounds__(256, 2) void decode_replay_elements_kernel(const DecReplayArgs a) {
  constexpr int NDC = DP / 16, CPR = DP / 8, TILE = 64 * DP, CH = DP > 128 ? 32 : 64;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][TILE];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_q[CH * DP * 2];
  __shared__ __attribute__((aligned(16))) float lse[CH], weight[CH];
  __shared__ int place[CH];                 // row's index on the path
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int hkv = (int)blockIdx.y, b = (int)blockIdx.z, bh = b * (int)gridDim.y + hkv;
  const int n = __builtin_amdgcn_readfirstlane(min(max(a.length[bh], 0), a.C));
  const int nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.A), share = dec_split<4>(tiles, a.S);
  const int t0 = (int)blockIdx.x * share, t1 = min(tiles, t0 + share);
  if (t0 >= t1) return;
  {
    const int na = dec_path_len(a, b), rows = a.G * na;
    const DecI32In path = a.path ? a.path + (long long)b * a.A : (DecI32In) nullptr;
    const float keep = fast_exp2(-a.decay_log2 * (float)na);

    const DecIn kc = a.kc + b * a.kcb + hkv * a.kch, kn = a.k + b * a.kb + hkv * a.kh, vn = a.v + b * a.vb + hkv * a.vh;
    for (int r0 = 0; r0 == 0 || r0 < rows; r0 += CH) {
      __syncthreads();                      // the rows before are done with
      for (int i = threadIdx.x; i < CH; i += 256) {
        const int r = r0 + i;
        float z = -kDecNegInf;              // no row: no weight
        int at = 0;
        if (r < rows) {
          const int g = r / na, node = path ? path[r - g * na] : r - g * na;
          at = r - g * na;
          z = a.lse[((long long)bh * a.G + g) * a.T + node];
          z = z == kDecNegInf ? -kDecNegInf : z;   // nothing visible: no weight
        }
        lse[i] = z;
        weight[i] = a.decay_log2 * (float)(at + 1 - na);
        place[i] = at;
      }
#pragma unroll 1
      for (int e = threadIdx.x; e < CH * CPR; e += 256) {
        const int r = r0 + e / CPR, ch = e % CPR;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (r < rows) {
          const int g = r / na, node = path ? path[r - g * na] : r - g * na;
          const DecIn qp = a.q + b * a.qb + (long long)(hkv * a.G + g) * a.qh + node * a.qn;
          x = dec_load8(qp, a.qc, ch, a.D);
        }
        *(u32x4*)(lds_q + dec_k_at<DP>(e / CPR, ch)) = x;
      }
      __syncthreads();
      const int rend = min(CH, rows - r0);

      for (int t = t0 + wv; t < t1; t += 4) {
        const bool tail = t >= nc;
        const int kb = tail ? (t - nc) * 32 : t * 32, krows = tail ? na : n;
        {
          const DecIn kp = tail ? kn : kc;
          const long long krs = tail ? a.kn64 : a.kcn64, kcs = tail ? a.kd : a.kcd;
#pragma unroll 1
          for (int i = 0; i < NDC; ++i) {
            const int e = i * 64 + lane, key = kb + e / CPR, ch = e % CPR;
            const int row = tail && path && key < krows ? path[key] : key;   // new rows in the path's order
            u32x4 x = {0u, 0u, 0u, 0u};
            if (key < krows) x = dec_load8(kp + row * krs, kcs, ch, a.D);
            *(u32x4*)(lds[wv] + dec_k_at<DP>(e / CPR, ch)) = x;
          }
        }
        dec_wave_order();
        u32x4 kf[NDC];
#pragma unroll
        for (int c = 0; c < NDC; ++c) kf[c] = dec_kfrag<DP>(lds[wv], 0, c);
        float sum = 0.f;
        for (int rt = 0; rt < rend; rt += 32) {
          // lanes hold keys; register i holds row rt + 8 (i / 4) + 4 hh + i % 4
          f32x16 x;
#pragma unroll
          for (int c = 0; c < NDC; ++c) x = c == 0 ? E::mfma(dec_kfrag<DP>(lds_q, rt, 0), kf[0], (f32x16){}) : E::mfma(dec_kfrag<DP>(lds_q, rt, c), kf[c], x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int rr = rt + 8 * (i >> 2) + 4 * hh + (i & 3);
            float p = fast_exp2(__builtin_fmaf(__builtin_fmaf(x[i], a.scale, -lse[rr]), 1.f / kLn2, weight[rr]));
            if (tail && place[rr] < kb + l32) p = 0.f;   // row i of the path sees new row u <= i
            if (lse[rr] == -kDecNegInf) p = 0.f;         // no row, whatever the key
            sum += p;
          }
        }
        dec_wave_order();
        sum = half_swap_sum(sum);
        if (hh) continue;
        const int key = kb + l32;
        if (!tail) {
          if (key < n) {
            const float w = a.norm ? a.norm[bh * a.norm_stride + key] : 1.f;
            const DecF32 to = a.imp_out + bh * a.impo_stride + key;
            *to = (r0 ? *to : a.imp[bh * a.imp_stride + key] * keep) + w * sum;
          }
        } else if (key < a.A) {
          float w = 0.f;
          if (key < na) {
            w = 1.f;
            if (a.norm) {
              const DecIn vp = vn + (path ? path[key] : key) * a.vn64;
              w = 0.f;
              for (int d = 0; d < a.D; ++d) w += fabsf(E::to_f32(vp[d * a.vd]));
            }
          }
          const DecF32 to = a.new_imp + (long long)bh * a.A + key;
          *to = (r0 ? *to : 0.f) + (key < na ? w * sum : 0.f);
        }
      }
    }
  }
}

#define FE_DEC_DIMS(X) X(64) X(96) X(128) X(192) X(256)
#define FE_DEC_ROW(DP, E, T)                                                                                            \
  {DP, T, (const void*)decode_few_kernel<E, DP>,                                                                        \
   {(const void*)decode_wide_kernel<E, DP, 4>, (const void*)decode_wide_kernel<E, DP, (DP > 128 ? 4 : 8)>},             \
   (const void*)decode_elements_kernel<E, DP>, (const void*)decode_join_kernel<E, DP>,                                  \
   {(const void*)decode_replay_elements_kernel<E, DP>, (const void*)decode_replay_kernel<E, DP>}},
#define FE_DEC_ROWS(DP) FE_DEC_ROW(DP, F16, FE_DTYPE_F16) FE_DEC_ROW(DP, BF16, FE_DTYPE_BF16)
// Kernels by tile dim: wide of four waves, and of eight where their registers allow it.
struct DecKernels {
  int dp, dtype;
  const void* few;
  const void* wide[2];
  const void* elements;
  const void* join;
  const void* replay[2];
};
const DecKernels kDecKernels[] = {FE_DEC_DIMS(FE_DEC_ROWS)};

const DecKernels& dec_kernels(int64_t D, int dtype) {
  for (const auto& e : kDecKernels)
    if (e.dp >= D && e.dtype == dtype) return e;
  return kDecKernels[0];
}

void append_decode_resources(std::string& out) {
  for (const auto& e : kDecKernels) {
    const void* fns[7] = {e.few, e.wide[0], e.wide[1], e.join, e.replay[1], e.elements, e.replay[0]};
    const char* names[7] = {"decode_few", "decode_wide4", "decode_wide8", "decode_join", "decode_replay", "decode_elements", "decode_replay_elements"};
    for (int i = 0; i < 7; ++i) {
      if (i == 2 && e.dp > 128) continue;
      hipFuncAttributes attr;
      if (hipFuncGetAttributes(&attr, fns[i]) != hipSuccess) continue;
      char buf[512];
      snprintf(buf, sizeof(buf),
               "{\"kernel\":\"%s<%s,%d>\",\"registers_per_thread\":%d,\"lds_static_bytes\":%zu,"
               "\"lds_dynamic_bytes\":0,\"scratch_bytes_per_thread\":%zu,\"max_threads_per_block\":%d},",
               names[i], e.dtype ? "bf16" : "fp16", e.dp, attr.numRegs, (size_t)attr.sharedSizeBytes,
               (size_t)attr.localSizeBytes, attr.maxThreadsPerBlock);
      out += buf;
    }
  }
}

namespace {

// 16-byte loads of rows: unit channel stride, channels in whole 16-byte chunks, every row on a 16-byte boundary, and
// row strides of 31 bits.
bool vec_ok(const void* p, const long long (&st)[4], int64_t B, int64_t H, int64_t N, int64_t D) {
  return D % 8 == 0 && st[3] == 1 && (uintptr_t)p % 16 == 0 && (B <= 1 || st[0] % 8 == 0) && (H <= 1 || st[1] % 8 == 0) &&
         (N <= 1 || (st[2] % 8 == 0 && st[2] <= 0x7fffffffLL));
}

int dec_check(const char* who, int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t C, int64_t D, int dtype, float scale,
              float decay) {
  const std::string w(who);
  if (B < 1 || Hq < 1 || Hkv < 1 || T < 1 || C < 1 || D < 1 || Hq % Hkv || D > 256 || T > kDecMaxTokens) {
    set_error(w + ": invalid shape (1 <= T <= 256, D <= 256, Hq a multiple of Hkv)");
    return FE_ERR_INVALID;
  }
  if (dtype != FE_DTYPE_F16 && dtype != FE_DTYPE_BF16) {
    set_error(w + ": dtype must be fp16 or bf16");
    return FE_ERR_INVALID;
  }
  if (!isfinite(scale) || !isfinite(decay) || decay < 0) {
    set_error(w + ": scale must be finite, recency_decay finite and nonnegative");
    return FE_ERR_INVALID;
  }
  // grid axes: KV heads, and batch rows times blocks of at least 32 rows
  if (C > (1LL << 30) || Hkv > 65535 || B > 65535 || B * Hkv > (1LL << 30) || Hq / Hkv > 32767 || B * ((Hq / Hkv * T + 31) / 32) > 65535) {
    set_error(w + ": sizes exceed the supported range");
    return FE_ERR_UNSUPPORTED;
  }
  return FE_OK;
}

int dec_strides(const char* who, const int64_t* const* in, long long (*out)[4], int count) {
  for (int i = 0; i < count; ++i) {
    if (!in[i]) {
      set_error(std::string(who) + ": null stride array");
      return FE_ERR_INVALID;
    }
    for (int j = 0; j < 4; ++j) {
      if (in[i][j] < 0) {
        set_error(std::string(who) + ": negative strides are not supported");
        return FE_ERR_INVALID;
      }
      out[i][j] = in[i][j];
    }
  }
  return FE_OK;
}

// Whether the heads of a launch share `blocks` blocks by their lengths, which a block has to read first (0.5 us). Heads of
// one batch row mostly are of one length, and without that launches whose tiles all have a block of their own (`need`)
// gain nothing. Paths of 6 over eight rows of 18432 to 32768: 51.7 us without, 43.9 with; trees of 61 tokens over two rows
// of 32768 and 24576 82 and 77.6; of 64 tokens over eight equal rows 54.8 and 55.4.
bool dec_shared(bool wide, int64_t B, int64_t BH, int64_t blocks, int64_t need) {
  return (wide || (B > 1 && blocks < need)) && BH <= 128 && 2 * BH <= blocks;
}

// How an attention launch is laid out; the same for the workspace's size and the call.
struct DecPlan {
  int kind;                    // 0: elements, 1: few, 2: wide
  int waves, RB, RS, S;        // waves of a wide block; row blocks of a head, rows of one, splits
  int NB;                      // blocks (of each row block) that the heads of a wide launch share, or 0
  size_t o, ml, heads, logits, bytes; // offsets
};
DecPlan dec_plan(int64_t B, int64_t BH, int64_t R, int64_t C, int64_t T, int64_t DP, bool vec, bool weights) {
  DecPlan p = {};
  const int64_t RT = (R + 31) / 32;
  p.kind = !vec ? 0 : R <= kDecFewRows ? 1 : 2;
  // eight waves, two on a SIMD, where their registers and rows suffice: 64 rows of 32 heads over 8192 rows 35.4 us with
  // four and 39.1 with eight, 128 rows 41.8 and 42.7; 256 rows of 64 heads over 4096 76 and 67
  p.waves = DP > 128 || RT <= 4 ? 4 : 8;
  p.RB = (int)(p.kind == 2 ? (RT + p.waves - 1) / p.waves : RT);
  p.RS = (int)(p.kind == 2 ? 32 * ((RT + p.RB - 1) / p.RB) : p.kind == 1 ? 16 : 32);
  // as many blocks as the card holds at once, of at least a tile a wave
  const int64_t KT = p.kind == 2 ? 64 : 32, tiles = (C + KT - 1) / KT + (T + KT - 1) / KT;
  const int64_t resident = DP > 128 || (p.kind == 2 && p.waves == 8) ? 256 : 512;
  p.S = (int)std::max<int64_t>(1, std::min(resident / (BH * p.RB), (tiles + 3) / 4));
  const int64_t need = BH * (p.kind == 2 ? tiles : (tiles + 3) / 4);
  if (p.kind != 0 && dec_shared(p.kind == 2, B, BH, resident / p.RB, need)) p.NB = (int)std::min(resident / p.RB, need);
  auto area = [&](size_t elems) {
    const size_t at = p.bytes;
    p.bytes += (elems * 4 + 255) / 256 * 256;
    return at;
  };
  const size_t slots = p.NB ? (size_t)p.NB * p.RB : (size_t)BH * p.RB * (p.kind == 2 ? 1 : p.S);
  p.o = area(slots * p.RS * DP);
  p.ml = area(slots * p.RS * 2);
  p.heads = area(p.kind == 2 || p.NB ? 2 * BH : 0);
  p.logits = p.bytes;
  if (weights && R <= kDecLogitRows) area((size_t)BH * ((C + 31) / 32 + (T + 31) / 32) * R * 32);
  return p;
}

template <typename A>
int dec_launch(const char* who, const void* fn, dim3 grid, dim3 block, A& a, hipStream_t stream) {
  void* args[] = {&a};
  hipError_t err = hipLaunchKernel(fn, grid, block, args, 0, stream);
  if (err != hipSuccess) {
    set_error(std::string(who) + ": launch: " + hipGetErrorString(err));
    return FE_ERR_HIP;
  }
  return FE_OK;
}

template <typename P, typename Q>
void dec_set(P& to, Q* from) { to = (P)(uintptr_t)from; }

// A negative scale runs as |scale| on -Q, a zero one as 1 on zeros (a masked logit, -inf, times a zero scale would be
// NaN).
void dec_scale(DecArgs& a, float scale) {
  a.qand = scale == 0.f ? 0u : ~0u;
  a.qxor = scale < 0.f ? 0x80008000u : 0u;
  a.scale_log2 = scale == 0.f ? 1.f : (float)(fabs((double)scale) * 1.4426950408889634);
}

// st: strides of q, k, v and the K cache; a's path, lse, importance and norms set by the caller.
int dec_replay(const char* who, const DecKernels& kn, DecReplayArgs& a, const void* q, const void* k, const void* v, const void* k_cache,
               const int32_t* length, const long long (*st)[4], int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t A, int64_t C,
               int64_t D, float scale, float decay, hipStream_t stream) {
  const bool vec = vec_ok(q, st[0], B, Hq, T, D) && vec_ok(k, st[1], B, Hkv, T, D) && vec_ok(v, st[2], B, Hkv, T, D) &&
                   vec_ok(k_cache, st[3], B, Hkv, C, D);
  dec_set(a.q, q);
  dec_set(a.k, k);
  dec_set(a.v, v);
  dec_set(a.kc, k_cache);
  dec_set(a.length, length);
  a.qb = st[0][0], a.qh = st[0][1], a.qn = st[0][2], a.qc = st[0][3];
  a.kb = st[1][0], a.kh = st[1][1], a.kn = (u32)st[1][2], a.kn64 = st[1][2], a.kd = st[1][3];
  a.vb = st[2][0], a.vh = st[2][1], a.vn = (u32)st[2][2], a.vn64 = st[2][2], a.vd = st[2][3];
  a.kcb = st[3][0], a.kch = st[3][1], a.kcn = (u32)st[3][2], a.kcn64 = st[3][2], a.kcd = st[3][3];
  a.T = (int)T;
  a.C = (int)C;
  a.D = (int)D;
  a.G = (int)(Hq / Hkv);
  a.A = (int)A;
  a.scale = scale;
  a.decay_log2 = (float)((double)decay * 1.4426950408889634);
  // as many blocks as the card holds at once, of at least a tile a wave
  const int64_t tiles = (C + 31) / 32 + (A + 31) / 32;
  a.S = (int)std::max<int64_t>(1, std::min<int64_t>((kn.dp > 128 ? 256 : 512) / (B * Hkv), vec && a.G * A > 64 ? tiles : (tiles + 3) / 4));
  a.Hkv = (int)Hkv;
  a.BH = (int)(B * Hkv);
  const int64_t blocks = kn.dp > 128 ? 256 : 512;
  if (vec && dec_shared(false, B, B * Hkv, blocks, B * Hkv * (a.G * A > 64 ? tiles : (tiles + 3) / 4))) a.NB = (int)blocks;
  const dim3 grid = a.NB ? dim3((unsigned)a.NB) : dim3((unsigned)a.S, (unsigned)Hkv, (unsigned)B);
  return dec_launch(who, kn.replay[vec], grid, dim3(256), a, stream);
}

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" size_t fe_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t C, int64_t D, int weights) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || T < 1 || C < 1 || D < 1 || D > 256 || T > kDecMaxTokens || B > 65535 || Hkv > 65535 ||
      B * Hkv > (1LL << 30) || Hq / Hkv > 32767 || C > (1LL << 30) || B * ((Hq / Hkv * T + 31) / 32) > 65535)
    return 0;
  const int64_t dp = dec_kernels(D, 0).dp;
  return std::max(dec_plan(B, B * Hkv, Hq / Hkv * T, C, T, dp, false, weights != 0).bytes,
                  dec_plan(B, B * Hkv, Hq / Hkv * T, C, T, dp, true, weights != 0).bytes);
}

extern "C" int fe_decode_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache,
                                   const int32_t* length, const uint8_t* tree, int64_t tree_batch_stride, void* out, float* lse,
                                   const float* importance, int64_t importance_stride, const float* value_norm,
                                   int64_t value_norm_stride, float* importance_out, int64_t importance_out_stride,
                                   float* new_importance, int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t C, int64_t D,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* k_cache_strides, const int64_t* v_cache_strides, int dtype, float scale,
                                   float recency_decay, void* workspace, size_t workspace_bytes, void* hip_stream) {
  static const char* who = "fe_decode_attention";
  clear_error();
  if (int rc = dec_check(who, B, Hq, Hkv, T, C, D, dtype, scale, recency_decay)) return rc;
  if (!q || !k || !v || !k_cache || !v_cache || !length || !out || !lse || (importance && (!importance_out || !new_importance))) {
    set_error(std::string(who) + ": null pointer argument");
    return FE_ERR_INVALID;
  }
  if (tree_batch_stride < 0 || (importance && (importance_stride < C || importance_out_stride < C || (value_norm && value_norm_stride < C)))) {
    set_error(std::string(who) + ": invalid row stride");
    return FE_ERR_INVALID;
  }
  const int64_t* in[5] = {q_strides, k_strides, v_strides, k_cache_strides, v_cache_strides};
  long long st[5][4];
  if (int rc = dec_strides(who, in, st, 5)) return rc;
  const DecKernels& kn = dec_kernels(D, dtype);
  const size_t need = fe_decode_workspace_bytes(B, Hq, Hkv, T, C, D, importance != nullptr);
  if (!workspace || workspace_bytes < need) {
    set_error(std::string(who) + ": workspace too small; need " + std::to_string(need) + " bytes");
    return FE_ERR_WORKSPACE;
  }
  if ((uintptr_t)workspace % 16 || (uintptr_t)out % 8) {
    set_error(std::string(who) + ": workspace must lie on a 16-byte boundary, out on an 8-byte one");
    return FE_ERR_INVALID;
  }
  const bool vec = vec_ok(q, st[0], B, Hq, T, D) && vec_ok(k, st[1], B, Hkv, T, D) && vec_ok(v, st[2], B, Hkv, T, D) &&
                   vec_ok(k_cache, st[3], B, Hkv, C, D) && vec_ok(v_cache, st[4], B, Hkv, C, D);
  const int64_t BH = B * Hkv, R = Hq / Hkv * T;
  const DecPlan p = dec_plan(B, BH, R, C, T, kn.dp, vec, importance != nullptr);
  const bool logits = importance && R <= kDecLogitRows;
  char* ws = (char*)workspace;
  hipStream_t stream = (hipStream_t)hip_stream;
  DecArgs a = {};
  dec_set(a.q, q);
  dec_set(a.k, k);
  dec_set(a.v, v);
  dec_set(a.kc, k_cache);
  dec_set(a.vc, v_cache);
  dec_set(a.length, length);
  dec_set(a.tree, tree);
  dec_set(a.part_o, ws + p.o);
  dec_set(a.part_ml, ws + p.ml);
  if (logits) dec_set(a.logits, ws + p.logits);
  a.qb = st[0][0], a.qh = st[0][1], a.qn = st[0][2], a.qc = st[0][3];
  a.kb = st[1][0], a.kh = st[1][1], a.kn = (u32)st[1][2], a.kn64 = st[1][2], a.kd = st[1][3];
  a.vb = st[2][0], a.vh = st[2][1], a.vn = (u32)st[2][2], a.vn64 = st[2][2], a.vd = st[2][3];
  a.kcb = st[3][0], a.kch = st[3][1], a.kcn = (u32)st[3][2], a.kcn64 = st[3][2], a.kcd = st[3][3];
  a.vcb = st[4][0], a.vch = st[4][1], a.vcn = (u32)st[4][2], a.vcn64 = st[4][2], a.vcd = st[4][3];
  a.tree_stride = tree_batch_stride;
  a.T = (int)T;
  a.C = (int)C;
  a.D = (int)D;
  a.R = (int)R;
  a.RB = p.RB;
  a.RS = p.RS;
  a.S = p.S;
  a.Hkv = (int)Hkv;
  a.BH = (int)BH;
  a.NB = p.NB;
  if (p.kind == 2 || p.NB) dec_set(a.heads, ws + p.heads);
  a.max_tiles = (int)((C + 31) / 32 + (T + 31) / 32);
  dec_scale(a, scale);
  if (p.kind == 1) a.scale_log2 = (float)((double)scale * 1.4426950408889634);   // masks after the scale
  const void* fn = p.kind == 0 ? kn.elements : p.kind == 1 ? kn.few : kn.wide[p.waves == 8];
  const dim3 grid = p.NB ? dim3((unsigned)p.NB, (unsigned)p.RB) : p.kind == 2 ? dim3((unsigned)BH, (unsigned)p.RB) : dim3((unsigned)p.S, (unsigned)Hkv, (unsigned)(B * p.RB));
  if (int rc = dec_launch(who, fn, grid, dim3(p.kind == 2 ? 64 * p.waves : 256), a, stream)) return rc;

  DecJoinArgs o = {};
  o.part_o = (DecF32In)a.part_o;
  o.part_ml = (DecF32In)a.part_ml;
  o.logits = (DecF32In)a.logits;
  o.length = a.length;
  o.heads = (DecI32In)a.heads;
  dec_set(o.out, out);
  dec_set(o.lse, lse);
  dec_set(o.imp, importance);
  dec_set(o.norm, value_norm);
  dec_set(o.imp_out, importance_out);
  dec_set(o.new_imp, new_importance);
  o.v = a.v;
  o.imp_stride = importance_stride;
  o.norm_stride = value_norm_stride;
  o.impo_stride = importance_out_stride;
  o.vb = a.vb;
  o.vh = a.vh;
  o.vn = a.vn64;
  o.vd = a.vd;
  o.T = a.T;
  o.C = a.C;
  o.D = a.D;
  o.R = a.R;
  o.RB = a.RB;
  o.RS = a.RS;
  o.S = a.S;
  o.max_tiles = a.max_tiles;
  o.decay_log2 = (float)((double)recency_decay * 1.4426950408889634);
  // all of a block's groups of threads on a row where they have slots enough, else one on each (256 rows of 64 heads in 4
  // slots each: 51.0 us in all; all on a row 63.0)
  const int groups = 256 / (kn.dp / 4);
  o.rows = 2 * (p.NB ? p.NB / BH : p.kind == 2 ? 1 : p.S) > groups ? 1 : groups;
  o.out_blocks = (int)((R + o.rows - 1) / o.rows);
  const int64_t per = logits ? std::min<int64_t>((a.max_tiles + 7) / 8, std::max<int64_t>(1, kDecJoinBlocks / BH)) : 0;
  if (int rc = dec_launch(who, kn.join, dim3((unsigned)(o.out_blocks + per), (unsigned)Hkv, (unsigned)B), dim3(256), o, stream)) return rc;
  if (!importance || logits) return FE_OK;
  DecReplayArgs r = {};
  r.lse = (DecF32In)o.lse;
  r.imp = o.imp;
  r.norm = o.norm;
  r.imp_out = o.imp_out;
  r.new_imp = o.new_imp;
  r.imp_stride = importance_stride;
  r.norm_stride = value_norm_stride;
  r.impo_stride = importance_out_stride;
  return dec_replay(who, kn, r, q, k, v, k_cache, length, st, B, Hq, Hkv, T, T, C, D, scale, recency_decay, stream);
}

extern "C" int fe_replay_path(const void* q, const void* k, const void* v, const void* k_cache, const int32_t* length,
                              const float* lse, const int32_t* path, const float* importance, int64_t importance_stride,
                              const float* value_norm, int64_t value_norm_stride, float* importance_out,
                              int64_t importance_out_stride, float* new_importance, int64_t B, int64_t Hq, int64_t Hkv,
                              int64_t T, int64_t A, int64_t C, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                              const int64_t* v_strides, const int64_t* k_cache_strides, int dtype, float scale,
                              float recency_decay, void* hip_stream) {
  static const char* who = "fe_replay_path";
  clear_error();
  if (int rc = dec_check(who, B, Hq, Hkv, T, C, D, dtype, scale, recency_decay)) return rc;
  if (A < 1 || A > T || (!path && A != T)) {
    set_error(std::string(who) + ": a path has 1 to T nodes (T without a path)");
    return FE_ERR_INVALID;
  }
  if (!q || !k || !v || !k_cache || !length || !lse || !importance || !importance_out || !new_importance) {
    set_error(std::string(who) + ": null pointer argument");
    return FE_ERR_INVALID;
  }
  if (importance_stride < C || importance_out_stride < C || (value_norm && value_norm_stride < C)) {
    set_error(std::string(who) + ": invalid row stride");
    return FE_ERR_INVALID;
  }
  const int64_t* in[4] = {q_strides, k_strides, v_strides, k_cache_strides};
  long long st[4][4];
  if (int rc = dec_strides(who, in, st, 4)) return rc;
  DecReplayArgs a = {};
  dec_set(a.lse, lse);
  dec_set(a.path, path);
  dec_set(a.imp, importance);
  a.imp_stride = importance_stride;
  dec_set(a.norm, value_norm);
  a.norm_stride = value_norm_stride;
  dec_set(a.imp_out, importance_out);
  a.impo_stride = importance_out_stride;
  dec_set(a.new_imp, new_importance);
  return dec_replay(who, dec_kernels(D, dtype), a, q, k, v, k_cache, length, st, B, Hq, Hkv, T, A, C, D, scale, recency_decay,
                    (hipStream_t)hip_stream);
}
