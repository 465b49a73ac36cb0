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
//   decode_rows_kernel     up to 32 query rows r = g * T + t of a group: each wave takes 32 keys at a time for all of
//                          them, S^T = K Q^T and O^T = V^T P^T on MFMA, with the rows' running maximum and sum
//   decode_wide_kernel     more rows: each wave holds 32 of them, the block's waves share tiles of 64 keys in LDS
//   decode_join_kernel     joins the splits of the keys: out and lse; and, where the first kernel left its logits
//                          (few rows), the importance, whose probabilities need the joined lse
//   decode_replay_kernel   the importance otherwise: S = Q K^T for the rows that stay, lanes holding keys, so that a
//                          key's sum over the rows is in-lane: p = exp2(x log2e - bias), the bias holding lse and w
//
// Lengths are known on the device only, and differ from head to head, so a launch has as many blocks as the card
// holds at once, and each takes an equal share of all tiles of all heads, in order (dec_share).
#include <math.h>
#include <algorithm>
#include <string>

#include "fe_attn.h"
#include "fe_internal.h"
#include "../../include/flash_evict.h"

namespace fe {

typedef __attribute__((address_space(3))) void* dec_lds_ptr;
typedef short dec_s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) dec_s16x4 dec_lds_s16x4;

constexpr int kDecMaxTokens = 256;   // new tokens of a call
// Rows of a group up to which the attention leaves its logits for the importance: 8 bytes a row and key, written and
// read, against the 2 D of reading K again.
constexpr int kDecLogitRows = 16;

struct DecArgs {
  const u16* q;
  const u16* k;            // new rows
  const u16* v;
  const u16* kc;           // cache
  const u16* vc;
  const int* length;       // [B * Hkv]
  const unsigned char* tree;   // [T, T] or [B, T, T], or null: causal
  const int* path;         // [B, A] nodes of the accepted path, or null: all T
  u16* out;                // [B, Hq, T, D]
  float* lse;              // [B, Hq, T]
  const float* lse_in;     // replay
  const float* imp;        // [B * Hkv] rows of imp_stride
  const float* norm;
  float* imp_out;
  float* new_imp;          // [B * Hkv, A]
  float* part_o;           // [slot][32 * RW][DP]: normalised partial outputs
  float* part_ml;          // [slot][2][32 * RW]: maximum (log2 units), sum
  int* seg;                // [segment][2]: first and last slot
  float* logits;           // [B * Hkv][tile][R][32] in log2 units, or null
  long long qs[4], ks[4], vs[4], kcs[4], vcs[4];
  long long imp_stride, norm_stride, impo_stride, tree_stride;
  int T, C, D, G, Hkv, BH, A;
  int R, RB, RW;           // rows of a group; segments of a group, 32-row tiles of a segment
  int nb;                  // blocks that share the tiles
  int max_tiles;           // tiles of 32 keys of a full cache and T new rows
  int join_blocks, join_split;   // decode_join_kernel: blocks of the output; 32-lane groups that share a row
  u32 qand, qxor;          // Q's sign for a negative scale, Q's zeros for a zero one
  float scale_log2, decay_log2;
};

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kDecNegInf = -__builtin_huge_valf();

// Rows of the (b, j) cache, within the tensor whatever the caller's length says.
__device__ __forceinline__ int dec_len(const DecArgs& a, int bh) { return min(max(a.length[bh], 0), a.C); }

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
template <int VEC>
__device__ __forceinline__ u32x4 dec_load8(const u16* row, long long cs, int ch, int D) {
  return load8(row, cs, 8 * ch, D, VEC);
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

// The tiles of KT keys of a head: its cache's, then those of `fresh` new rows.
template <int KT>
__device__ __forceinline__ int dec_tiles(int n, int fresh) { return (n + KT - 1) / KT + (fresh + KT - 1) / KT; }

__device__ __forceinline__ long long dec_lane64(long long x, int lane) {
  const u32 lo = __builtin_amdgcn_readlane((u32)x, lane), hi = __builtin_amdgcn_readlane((u32)((unsigned long long)x >> 32), lane);
  return (long long)(((unsigned long long)hi << 32) | lo);
}

// Block blockIdx.x's share [pos, hi) of the W tiles of all segments, numbered head by head and, within a head,
// segment by segment of all its tiles; the head that holds pos and the head's first tile. Only as many blocks share
// as there are PER tiles for each, so no block between two others is without a tile. Every wave computes it.
struct DecShare {
  long long pos, hi, base;
  int bh;
};
template <int KT, int PER>
__device__ __forceinline__ DecShare dec_share(const DecArgs& a, int segs, int fresh) {
  const int lane = threadIdx.x & 63;
  long long W = 0, first = 0;
  for (int c0 = 0; c0 < a.BH; c0 += 64) {
    long long x = c0 + lane < a.BH ? (long long)segs * dec_tiles<KT>(dec_len(a, c0 + lane), fresh) : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const long long y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    if (c0 == 0) first = x;
    W += dec_lane64(x, 63);
  }
  DecShare s;
  const long long nb = min((long long)a.nb, (W + PER - 1) / PER);
  s.pos = s.hi = 0;
  if ((long long)blockIdx.x < nb) {
    s.pos = W * (long long)blockIdx.x / nb;
    s.hi = W * ((long long)blockIdx.x + 1) / nb;
  }
  s.base = 0;
  s.bh = 0;
  for (int c0 = 0; c0 < a.BH; c0 += 64) {
    long long x = first;
    if (c0) {
      x = c0 + lane < a.BH ? (long long)segs * dec_tiles<KT>(dec_len(a, c0 + lane), fresh) : 0;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const long long y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
    }
    const unsigned long long past = __ballot(s.base + x > s.pos);
    if (past) {
      const int at = __ffsll(past) - 1;
      s.bh = c0 + at;
      if (at) s.base += dec_lane64(x, at - 1);
      break;
    }
    s.base += dec_lane64(x, 63);
  }
  return s;
}

// Which of a lane's 16 keys of 32 from kb (bit i: key kb + 8 (i / 4) + 4 hh + i % 4) query token tq sees, among the
// cache's rows (fresh false) or the new ones.
__device__ __forceinline__ u32 dec_visible(const DecArgs& a, int b, int tq, int kb, int rows, bool fresh) {
  const int k0 = kb + 4 * (int)((threadIdx.x >> 5) & 1);
  const unsigned char* row = a.tree + b * a.tree_stride + tq * a.T;
  u32 bits = 0;
#pragma unroll 1
  for (int i = 0; i < 16; i += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = k0 + 2 * i + j;
      bool see = key < rows;
      if (fresh) see = see && (a.tree ? row[see ? key : 0] != 0 : key <= tq);
      bits |= (see ? 1u : 0u) << (i + j);
    }
  }
  return bits;
}

// Where a tile of KT keys lies: tile t of nc of the cache, then of the new rows.
struct DecTile {
  const u16 *k, *v;
  long long krs, vrs;
  int kb, rows;
  bool tail;
};
template <int KT>
__device__ __forceinline__ DecTile dec_tile(const DecArgs& a, int b, int hkv, int n, int nc, int fresh, int t) {
  DecTile x;
  x.tail = t >= nc;
  x.kb = (x.tail ? t - nc : t) * KT;
  x.rows = x.tail ? fresh : n;
  x.krs = x.tail ? a.ks[2] : a.kcs[2];
  x.vrs = x.tail ? a.vs[2] : a.vcs[2];
  x.k = x.tail ? a.k + b * a.ks[0] + hkv * a.ks[1] : a.kc + b * a.kcs[0] + hkv * a.kcs[1];
  x.v = x.tail ? a.v + b * a.vs[0] + hkv * a.vs[1] : a.vc + b * a.vcs[0] + hkv * a.vcs[1];
  return x;
}

// Chunk i of NT threads' 16-byte chunks of KT rows from row kb on (zeros past `rows` and past channel D): thread tid has
// chunk e = i * NT + tid in row order. Where a row's chunks divide the threads, a thread's channel is the same in each.
template <int DP, int KT, int NT, int NL>
__device__ __forceinline__ void dec_load_rows(const u16* p, long long rs, int kb, int rows, int D, int tid, u32x4 (&x)[NL]) {
  constexpr int CPR = DP / 8;
  if constexpr (NT % CPR == 0) {
    const int key = tid / CPR, ch = 8 * (tid % CPR);
    const u16* lp = p + key * rs + ch;
    const bool in = ch < D;
    if (kb + KT <= rows) {
#pragma unroll
      for (int i = 0; i < NL; ++i) x[i] = in ? *(const u32x4*)(lp + (long long)(kb + i * (NT / CPR)) * rs) : (u32x4){0u, 0u, 0u, 0u};
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        x[i] = in && kb + key + i * (NT / CPR) < rows ? *(const u32x4*)(lp + (long long)(kb + i * (NT / CPR)) * rs) : (u32x4){0u, 0u, 0u, 0u};
    }
  } else {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = i * NT + tid, key = e / CPR, ch = 8 * (e % CPR);
      const bool ok = kb + key < rows && ch < D && (KT * CPR % NT == 0 || key < KT);
      x[i] = ok ? *(const u32x4*)(p + (long long)(kb + key) * rs + ch) : (u32x4){0u, 0u, 0u, 0u};
    }
  }
}

// The segment's place in the tables, and its first and last slot, by the blocks that hold its ends. A block's
// segments follow each other, so block + segment numbers every (block, segment) pair apart.
__device__ __forceinline__ int dec_slot(const DecArgs& a, int seg, bool head, bool end) {
  const int slot = (int)blockIdx.x + seg;
  if (threadIdx.x == 0) {
    if (head) a.seg[2 * seg] = slot;
    if (end) a.seg[2 * seg + 1] = slot;
  }
  return slot;
}

// What bounds it: HBM. Few rows leave the matrix and vector units mostly idle, so every wave keeps the next 32 keys'
// K and V on the way to registers while it works on these.
template <typename E, int DP, int VEC>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void decode_rows_kernel(const DecArgs a) {
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

  DecShare sh = dec_share<32, 4>(a, a.RB, a.T);
  while (sh.pos < sh.hi) {
    const int bh = sh.bh, b = bh / a.Hkv, hkv = bh - b * a.Hkv;
    const int n = dec_len(a, bh);
    const int nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.T);
    const int rb = (int)((sh.pos - sh.base) / tiles), t0 = (int)((sh.pos - sh.base) - (long long)rb * tiles);
    const int t1 = (int)min((long long)tiles, t0 + (sh.hi - sh.pos));
    sh.pos += t1 - t0;
    if (sh.pos - sh.base == (long long)a.RB * tiles) {
      sh.base = sh.pos;
      ++sh.bh;
    }

    const int r = rb * 32 + l32;         // this lane's query row
    const bool rv = r < a.R;
    const int g = rv ? r / a.T : 0, tq = rv ? r - g * a.T : 0;
    u32x4 qf[NDC];
    {
      const u16* qp = a.q + b * a.qs[0] + (hkv * a.G + g) * a.qs[1] + tq * a.qs[2];
#pragma unroll
      for (int c = 0; c < NDC; ++c) {
        qf[c] = rv ? (dec_load8<VEC>(qp, a.qs[3], 2 * c + hh, a.D) & a.qand) ^ a.qxor : (u32x4){0u, 0u, 0u, 0u};
        if (!VEC) __builtin_amdgcn_sched_barrier(0);   // element loads: one chunk's addresses at a time
      }
    }
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = (f32x16){};
    float m = kDecNegInf, l = 0.f, lr = 0.f;   // sums of the probabilities, and of these as rounded for the product

    u32x4 kx[VEC ? NDC : 1], vx[VEC ? NDC : 1];
    auto load = [&](int t) __attribute__((always_inline)) {
      const DecTile at = dec_tile<32>(a, b, hkv, n, nc, a.T, t);
      dec_load_rows<DP, 32, 64>(at.k, at.krs, at.kb, at.rows, a.D, lane, kx);
      dec_load_rows<DP, 32, 64>(at.v, at.vrs, at.kb, at.rows, a.D, lane, vx);
    };
    if (VEC && t0 + wv < t1) load(t0 + wv);
    for (int t = t0 + wv; t < t1; t += 4) {
      const DecTile at = dec_tile<32>(a, b, hkv, n, nc, a.T, t);
      const bool tail = at.tail;
      const int kb = at.kb, rows = at.rows;
      const long long vcs = tail ? a.vs[3] : a.vcs[3];
      // keys of the tail whose value has an infinity or a NaN: 0 * inf would reach the rows that do not see
      // them, so their values are taken out of the product and added to the rows that do
      u32 odd = 0;
      if (VEC) {
#pragma unroll
        for (int i = 0; i < NDC; ++i) {
          const int e = i * 64 + lane;
          *(u32x4*)(kt + dec_k_at<DP>(e / CPR, e % CPR)) = kx[i];
          *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = vx[i];
        }
        if (tail) {
#pragma unroll
          for (int i = 0; i < NDC; ++i)
            for (unsigned long long bl = __ballot(dec_nonfinite<E>(vx[i])); bl; bl &= bl - 1) odd |= 1u << ((i * 64 + __ffsll(bl) - 1) / CPR);
        }
        if (t + 4 < t1) load(t + 4);
      } else {
        const long long kcs = tail ? a.ks[3] : a.kcs[3];
#pragma unroll 1
        for (int i = 0; i < NDC; ++i) {
          const int e = i * 64 + lane, row = kb + e / CPR, ch = e % CPR;
          const u32x4 x = row < rows ? dec_load8<VEC>(at.k + row * at.krs, kcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
          *(u32x4*)(kt + dec_k_at<DP>(e / CPR, ch)) = x;
          __builtin_amdgcn_sched_barrier(0);
          const u32x4 y = row < rows ? dec_load8<VEC>(at.v + row * at.vrs, vcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
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
        vis = dec_visible(a, b, tq, kb, rows, tail);
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
        float* lp = a.logits + (((long long)bh * a.max_tiles + t) * a.R + r) * 32 + 4 * hh;
#pragma unroll
        for (int i = 0; i < 4; ++i) *(f32x4*)(lp + 8 * i) = (f32x4){x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
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
          for (int ch = lane; ch < DP; ch += 64) row[ch] = ch < a.D ? E::to_f32(at.v[(kb + key) * at.vrs + ch * vcs]) : 0.f;
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
    const int slot = dec_slot(a, bh * a.RB + rb, t0 == 0, t1 == tiles);
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
      a.part_o[((long long)slot * 32 + row) * DP + ch] = lrt == 0.f ? 0.f : s * (1.f / lrt);
      if (ch == 0) {
        a.part_ml[slot * 64 + row] = mx;
        a.part_ml[slot * 64 + 32 + row] = lt;
      }
    }
    __syncthreads();                        // the next segment's tiles follow these reads
  }
}

// A wave holds 32 of the segment's rows; the block's waves share tiles of 64 keys, double-buffered, whose loads are on
// the way to registers during the tile before. A row keeps its reference maximum until a tile's probabilities could
// overflow (E::kMaxTileSum), as in the prefill kernels, so most tiles spend nothing on maxima and rescaling.
// What bounds it: vector work beside the products (an exponential a logit); at 256 rows a tile takes about as long as
// its bytes from HBM.
template <typename E, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP > 128 ? 1 : 2) void decode_wide_kernel(const DecArgs a) {
  constexpr int NDC = DP / 16, NDT = DP / 32, CPR = DP / 8, TILE = 128 * DP;   // bytes of 64 rows
  constexpr int NT = NW * 64, NL = (64 * CPR + NT - 1) / NT;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k[2][TILE], lds_v[2][TILE];
  __shared__ u32 s_odd[2][2];            // keys of a tile of new rows with a value that is not finite
  __shared__ float s_row[NW][DP];        // such a value, by each wave
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);

  DecShare sh = dec_share<64, 1>(a, a.RB, a.T);
  while (sh.pos < sh.hi) {
    const int bh = sh.bh, b = bh / a.Hkv, hkv = bh - b * a.Hkv;
    const int n = dec_len(a, bh);
    const int nc = (n + 63) / 64, tiles = dec_tiles<64>(n, a.T);
    const int rb = (int)((sh.pos - sh.base) / tiles), t0 = (int)((sh.pos - sh.base) - (long long)rb * tiles);
    const int t1 = (int)min((long long)tiles, t0 + (sh.hi - sh.pos));
    sh.pos += t1 - t0;
    if (sh.pos - sh.base == (long long)a.RB * tiles) {
      sh.base = sh.pos;
      ++sh.bh;
    }

    const int r = (rb * a.RW + wv) * 32 + l32;
    const bool live = wv < a.RW && (rb * a.RW + wv) * 32 < a.R;   // the wave has rows
    const bool rv = live && r < a.R;
    const int g = rv ? r / a.T : 0, tq = rv ? r - g * a.T : 0;
    u32x4 qf[NDC];
    {
      const u16* qp = a.q + b * a.qs[0] + (hkv * a.G + g) * a.qs[1] + tq * a.qs[2];
#pragma unroll
      for (int c = 0; c < NDC; ++c) qf[c] = rv ? (dec_load8<1>(qp, 1, 2 * c + hh, a.D) & a.qand) ^ a.qxor : (u32x4){0u, 0u, 0u, 0u};
    }
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = (f32x16){};
    float m = kDecNegInf, nm = 0.f, l = 0.f, lr = 0.f;   // lane-wise sums (half of a row's keys each)
    u32 ones2;
    asm volatile("s_mov_b32 %0, %1" : "=s"(ones2) : "i"(E::kOnes2));

    u32x4 kx[NL], vx[NL];
    auto load = [&](int t) __attribute__((always_inline)) {
      const DecTile at = dec_tile<64>(a, b, hkv, n, nc, a.T, t);
      dec_load_rows<DP, 64, NT>(at.k, at.krs, at.kb, at.rows, a.D, tid, kx);
      dec_load_rows<DP, 64, NT>(at.v, at.vrs, at.kb, at.rows, a.D, tid, vx);
    };
    auto store = [&](int t, int buf) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int e = i * NT + tid, key = e / CPR, ch = e % CPR;
        if (64 * CPR % NT == 0 || key < 64) {
          *(u32x4*)(lds_k[buf] + dec_k_at<DP>(key, ch)) = kx[i];
          *(u32x4*)(lds_v[buf] + dec_v_at<DP>(key, ch)) = vx[i];
        }
      }
      if (t >= nc) {
        if (tid < 2) s_odd[buf][tid] = 0u;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int key = (i * NT + tid) / CPR;
          if (dec_nonfinite<E>(vx[i])) atomicOr(&s_odd[buf][key >> 5], 1u << (key & 31));
        }
      }
    };
    load(t0);
    store(t0, t0 & 1);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int buf = t & 1;
      const bool tail = t >= nc;
      const int kb = tail ? (t - nc) * 64 : t * 64, rows = tail ? a.T : n;
      unsigned char* kt = lds_k[buf];
      unsigned char* vt = lds_v[buf];
      if (t + 1 < t1) load(t + 1);
      unsigned long long odd = 0;
      if (tail) {
        odd = ((unsigned long long)s_odd[buf][1] << 32) | s_odd[buf][0];
        if (odd) {
          for (int e = tid; e < 64 * CPR; e += NT)
            if ((odd >> (e / CPR)) & 1u) *(u32x4*)(vt + dec_v_at<DP>(e / CPR, e % CPR)) = (u32x4){0u, 0u, 0u, 0u};
          __syncthreads();
        }
      }
      if (live) {
        u32 vis[2] = {~0u, ~0u};
        const bool masked = tail || kb + 64 > rows;
        if (masked) {
          vis[0] = dec_visible(a, b, tq, kb, rows, tail);
          vis[1] = dec_visible(a, b, tq, kb + 32, rows, tail);
        }
        f32x16 x[2];                       // logits, then probabilities
        auto logits = [&]() __attribute__((always_inline)) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int c = 0; c < NDC; ++c)
              x[s] = c == 0 ? E::mfma(dec_kfrag<DP>(kt, 32 * s, 0), qf[0], (f32x16){}) : E::mfma(dec_kfrag<DP>(kt, 32 * s, c), qf[c], x[s]);
            if (masked) {
#pragma unroll
              for (int i = 0; i < 16; ++i) x[s][i] = (vis[s] >> i) & 1u ? x[s][i] : kDecNegInf;
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
          if (half_swap_max(over ? 1.f : 0.f) > 0.f && mx > m) {
            const float alpha = m == kDecNegInf ? 0.f : fast_exp2(m - mx);
            m = mx;
            nm = -mx;
            l *= alpha;
            lr *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
          }
          exponentials();
        }
        if (odd) {
          const u16* vp = a.v + b * a.vs[0] + hkv * a.vs[1];
#pragma unroll 1
          for (unsigned long long left = odd; left; left &= left - 1) {
            const int key = __ffsll(left) - 1;
            // the register and half that hold the key, where the lane's query sees it
            float mine = -1.f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (key == 32 * s + 8 * (i >> 2) + 4 * hh + (i & 3) && ((vis[s] >> i) & 1u)) mine = x[s][i];
            const float pk = half_swap_max(mine);      // probabilities are not negative
            const float nan = half_swap_max(mine != mine ? 1.f : 0.f);
            const float pr = nan > 0.f ? __builtin_nanf("") : pk;
            const bool sees = pk >= 0.f || nan > 0.f;
            const u16* row = vp + (long long)(kb + key) * a.vs[2];
            for (int ch = lane; ch < DP; ch += 64) s_row[wv][ch] = ch < a.D ? E::to_f32(row[ch]) : 0.f;
            dec_wave_order();
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float y = s_row[wv][32 * dt + 8 * (i >> 2) + 4 * hh + (i & 3)];
                if (sees) o[dt][i] += pr * y;
              }
            dec_wave_order();
          }
        }
        l += ls;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int c4 = 0; c4 < 2; ++c4) {
            u32x4 pf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              pf[i] = E::pack2(x[s][8 * c4 + 2 * i], x[s][8 * c4 + 2 * i + 1]);
              lr = E::sum2(pf[i], ones2, lr);
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] = E::mfma(dec_vfrag<DP>(vt, 32 * s + 16 * c4, dt), pf, o[dt]);
          }
      }
      if (t + 1 < t1) store(t + 1, buf ^ 1);
      __syncthreads();
    }

    const int slot = dec_slot(a, bh * a.RB + rb, t0 == 0, t1 == tiles);
    l = half_swap_sum(l);
    lr = half_swap_sum(lr);
    if (rv) {
      const float inv = lr == 0.f ? 0.f : 1.f / lr;
      const int row = wv * 32 + l32;
      float* po = a.part_o + ((long long)slot * a.RW * 32 + row) * DP;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(po + 32 * dt + 8 * i + 4 * hh) =
              (f32x4){o[dt][4 * i] * inv, o[dt][4 * i + 1] * inv, o[dt][4 * i + 2] * inv, o[dt][4 * i + 3] * inv};
      if (hh == 0) {
        a.part_ml[(long long)slot * 64 * a.RW + row] = m;
        a.part_ml[(long long)slot * 64 * a.RW + 32 * a.RW + row] = l;
      }
    }
  }
}

// Blocks below join_blocks: out = sum_s w_s O_s / sum w_s with w_s = l_s 2^(m_s - m), eight 32-lane groups a block,
// join_split of them (1 or 8) on each row. Later blocks, where there are logits: eight tiles of 32 keys of a head,
// importance_out and new_importance.
template <typename E, int DP>
__global__ __launch_bounds__(256) void decode_join_kernel(const DecArgs a) {
  constexpr int NV = (DP + 127) / 128;      // float4 of a lane
  __shared__ float sm[8][32], sl[8][32];
  __shared__ float bias[32];
  __shared__ f32x4 so[8][32 * NV];
  const int l32 = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int RS = a.RW * 32;                 // rows of a segment
  if ((int)blockIdx.x < a.join_blocks) {
    const int per = 8 / a.join_split, sub = grp % a.join_split;
    const long long gr = (long long)blockIdx.x * per + grp / a.join_split;   // row of all heads' rows
    const bool rv = gr < (long long)a.BH * a.R;
    const int bh = rv ? (int)(gr / a.R) : 0, r = rv ? (int)(gr - (long long)bh * a.R) : 0;
    const int sg = bh * a.RB + r / RS, row = r % RS;
    const int first = a.seg[2 * sg], count = rv ? a.seg[2 * sg + 1] - first + 1 : 0;
    const float* ml = a.part_ml + (long long)first * 2 * RS + row;
    float m = kDecNegInf;
    for (int s = l32; s < count; s += 32) m = fmaxf(m, ml[(long long)s * 2 * RS]);
#pragma unroll
    for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float ref = m == kDecNegInf ? 0.f : m;
    float l = 0.f;
    for (int s = l32; s < count; s += 32) l += ml[(long long)s * 2 * RS + RS] * fast_exp2(ml[(long long)s * 2 * RS] - ref);
#pragma unroll
    for (int d = 16; d; d /= 2) l += __shfl_xor(l, d);
    f32x4 acc[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) acc[v] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const float* po = a.part_o + ((long long)first * RS + row) * DP + 4 * l32;
#pragma unroll 4
    for (int s = sub; s < count; s += a.join_split) {
      // a split that this row sees nothing of has a weight of 0 and values of 0
      const float w = ml[(long long)s * 2 * RS + RS] * fast_exp2(ml[(long long)s * 2 * RS] - ref);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (128 * v + 4 * l32 < DP) acc[v] += w * *(const f32x4*)(po + (long long)s * RS * DP + 128 * v);
    }
    if (a.join_split > 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v) so[grp][v * 32 + l32] = acc[v];
      __syncthreads();
      if (sub) return;
      for (int i = 1; i < a.join_split; ++i)
#pragma unroll
        for (int v = 0; v < NV; ++v) acc[v] += so[grp + i][v * 32 + l32];
    }
    if (!rv) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int b = bh / a.Hkv, hkv = bh - b * a.Hkv, g = r / a.T, t = r - g * a.T;
    const long long at = ((long long)b * a.Hkv * a.G + hkv * a.G + g) * a.T + t;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = 128 * v + 4 * l32;
      const u32 w0 = E::pack2(acc[v][0] * inv, acc[v][1] * inv), w1 = E::pack2(acc[v][2] * inv, acc[v][3] * inv);
      u16* op = a.out + at * a.D + d;
      if (a.D % 4 == 0) {
        if (d < a.D) *(u32x2*)op = (u32x2){w0, w1};
      } else {
        const u16 h[4] = {(u16)w0, (u16)(w0 >> 16), (u16)w1, (u16)(w1 >> 16)};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < a.D) op[i] = h[i];
      }
    }
    if (l32 == 0) a.lse[at] = l == 0.f ? kDecNegInf : (m + fast_log2(l)) * kLn2;
    return;
  }

  // importance: a head's R <= kDecLogitRows rows are one segment
  const int blk = (int)blockIdx.x - a.join_blocks, bh = blk % a.BH, t = blk / a.BH * 8 + grp;
  const int b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  const int n = dec_len(a, bh), nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.T);
  if (blk / a.BH * 8 >= tiles) return;
  {
    const int first = a.seg[2 * bh], count = a.seg[2 * bh + 1] - first + 1;
    const float* ml = a.part_ml + (long long)first * 64 + l32;
    const bool rv = l32 < a.R;
    float m = kDecNegInf;
    for (int s = grp; s < count; s += 8) m = rv ? fmaxf(m, ml[s * 64]) : m;
    sm[grp][l32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, sm[i][l32]);
    const float ref = m == kDecNegInf ? 0.f : m;
    float l = 0.f;
    for (int s = grp; s < count; s += 8) l += rv ? ml[s * 64 + 32] * fast_exp2(ml[s * 64] - ref) : 0.f;
    sl[grp][l32] = l;
    __syncthreads();
    if (grp == 0) {
      l = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) l += sl[i][l32];
      // log2 of l and of w = 2^(-decay (T - 1 - t)); rows that see nothing give no weight
      bias[l32] = l == 0.f ? -kDecNegInf : ref + fast_log2(l) + a.decay_log2 * (float)(a.T - 1 - l32 % a.T);
    }
    __syncthreads();
  }
  if (t >= tiles) return;
  const float* lp = a.logits + ((long long)bh * a.max_tiles + t) * a.R * 32 + l32;
  float sum = 0.f;
#pragma unroll 4
  for (int r = 0; r < a.R; ++r) sum += fast_exp2(lp[r * 32] - bias[r]);
  if (t < nc) {
    const int key = t * 32 + l32;
    if (key < n) {
      const float old = a.imp[bh * a.imp_stride + key] * fast_exp2(-a.decay_log2 * (float)a.T);
      a.imp_out[bh * a.impo_stride + key] = old + (a.norm ? a.norm[bh * a.norm_stride + key] : 1.f) * sum;
    }
  } else {
    const int u = (t - nc) * 32 + l32;
    if (u < a.T) {
      float w = 1.f;
      if (a.norm) {
        const u16* vp = a.v + b * a.vs[0] + hkv * a.vs[1] + u * a.vs[2];
        w = 0.f;
        for (int d = 0; d < a.D; ++d) w += fabsf(E::to_f32(vp[d * a.vs[3]]));
      }
      a.new_imp[(long long)bh * a.T + u] = w * sum;
    }
  }
}

// Leading nodes of batch row b's path that name one of the T tokens.
__device__ __forceinline__ int dec_path_len(const DecArgs& a, int b) {
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

// Rows whose Q is in LDS at a time.
template <int DP>
constexpr int dec_replay_rows() { return DP > 128 ? 32 : 64; }

// What bounds it: reading K. A wave takes 32 keys at a time through its own LDS into registers, the next 32 on the
// way, against the rows' Q in LDS. More rows than that has room for take K again (from L2 mostly), adding to what
// the rows before left.
template <typename E, int DP, int VEC>
__global__ __launch_bounds__(256, 2) void decode_replay_kernel(const DecArgs a) {
  constexpr int NDC = DP / 16, CPR = DP / 8, TILE = 64 * DP, CH = dec_replay_rows<DP>();
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][TILE];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_q[CH * DP * 2];
  __shared__ __attribute__((aligned(16))) float bias[CH];
  __shared__ int place[CH];                 // row's index on the path
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  DecShare sh = dec_share<32, 4>(a, 1, a.A);
  while (sh.pos < sh.hi) {
    const int bh = sh.bh, b = bh / a.Hkv, hkv = bh - b * a.Hkv;
    const int n = dec_len(a, bh);
    const int nc = (n + 31) / 32, tiles = dec_tiles<32>(n, a.A);
    const int t0 = (int)(sh.pos - sh.base), t1 = (int)min((long long)tiles, t0 + (sh.hi - sh.pos));
    sh.pos += t1 - t0;
    if (t1 == tiles) {
      sh.base = sh.pos;
      ++sh.bh;
    }
    const int na = dec_path_len(a, b), rows = a.G * na;
    const int* path = a.path ? a.path + (long long)b * a.A : nullptr;
    const float keep = fast_exp2(-a.decay_log2 * (float)na);

    u32x4 kx[VEC ? NDC : 1];
    auto load = [&](int t) __attribute__((always_inline)) {
      if constexpr (VEC) dec_load_rows<DP, 32, 64>(a.kc + b * a.kcs[0] + hkv * a.kcs[1], a.kcs[2], t * 32, n, a.D, lane, kx);
    };
    for (int r0 = 0; r0 == 0 || r0 < rows; r0 += CH) {
      if (VEC && t0 + wv < min(t1, nc)) load(t0 + wv);
      __syncthreads();                      // the rows before are done with
      for (int i = threadIdx.x; i < CH; i += 256) {
        const int r = r0 + i;
        float bs = -kDecNegInf;
        int at = 0;
        if (r < rows) {
          const int g = r / na, node = path ? path[r - g * na] : r - g * na;
          at = r - g * na;
          const float z = a.lse_in[((long long)b * a.Hkv * a.G + hkv * a.G + g) * a.T + node];
          // nothing visible (lse = -inf): the row gives no weight
          if (z != kDecNegInf) bs = z * (1.f / kLn2) + a.decay_log2 * (float)(na - 1 - at);
        }
        bias[i] = bs;
        place[i] = at;
      }
#pragma unroll 1
      for (int e = threadIdx.x; e < CH * CPR; e += 256) {
        const int r = r0 + e / CPR, ch = e % CPR;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (r < rows) {
          const int g = r / na, node = path ? path[r - g * na] : r - g * na;
          x = (dec_load8<VEC>(a.q + b * a.qs[0] + (hkv * a.G + g) * a.qs[1] + node * a.qs[2], a.qs[3], ch, a.D) & a.qand) ^ a.qxor;
        }
        *(u32x4*)(lds_q + dec_k_at<DP>(e / CPR, ch)) = x;
      }
      __syncthreads();
      const int rend = min(CH, rows - r0);

      for (int t = t0 + wv; t < t1; t += 4) {
        const bool tail = t >= nc;
        const int kb = tail ? (t - nc) * 32 : t * 32, krows = tail ? na : n;
        if (VEC && !tail) {
#pragma unroll
          for (int i = 0; i < NDC; ++i) {
            const int e = i * 64 + lane;
            *(u32x4*)(lds[wv] + dec_k_at<DP>(e / CPR, e % CPR)) = kx[i];
          }
          if (t + 4 < min(t1, nc)) load(t + 4);
        } else {
          const u16* kp = tail ? a.k + b * a.ks[0] + hkv * a.ks[1] : a.kc + b * a.kcs[0] + hkv * a.kcs[1];
          const long long krs = tail ? a.ks[2] : a.kcs[2], kcs = tail ? a.ks[3] : a.kcs[3];
#pragma unroll 1
          for (int i = 0; i < NDC; ++i) {
            const int e = i * 64 + lane, key = kb + e / CPR, ch = e % CPR;
            const int row = tail && path && key < krows ? path[key] : key;   // new rows in the path's order
            const u32x4 x = key < krows ? dec_load8<VEC>(kp + row * krs, kcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
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
            float p = fast_exp2(x[i] * a.scale_log2 - bias[rr]);
            if (tail && place[rr] < kb + l32) p = 0.f;   // row i of the path sees new row u <= i
            if (bias[rr] == -kDecNegInf) p = 0.f;        // no row, whatever the key
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
            float* to = a.imp_out + bh * a.impo_stride + key;
            *to = (r0 ? *to : a.imp[bh * a.imp_stride + key] * keep) + w * sum;
          }
        } else if (key < a.A) {
          float w = 0.f;
          if (key < na) {
            w = 1.f;
            if (a.norm) {
              const u16* vp = a.v + b * a.vs[0] + hkv * a.vs[1] + (path ? path[key] : key) * a.vs[2];
              w = 0.f;
              for (int d = 0; d < a.D; ++d) w += fabsf(E::to_f32(vp[d * a.vs[3]]));
            }
          }
          float* to = a.new_imp + (long long)bh * a.A + key;
          *to = (r0 ? *to : 0.f) + (key < na ? w * sum : 0.f);
        }
      }
    }
  }
}

#define FE_DEC_DIMS(X) X(64) X(96) X(128) X(192) X(256)
#define FE_DEC_ROW(DP, E, T)                                                                                            \
  {DP, T, {(const void*)decode_rows_kernel<E, DP, 0>, (const void*)decode_rows_kernel<E, DP, 1>},                       \
   {(const void*)decode_wide_kernel<E, DP, 4>, (const void*)decode_wide_kernel<E, DP, (DP > 128 ? 4 : 8)>},              \
   (const void*)decode_join_kernel<E, DP>,                                                                              \
   {(const void*)decode_replay_kernel<E, DP, 0>, (const void*)decode_replay_kernel<E, DP, 1>}},
#define FE_DEC_ROWS(DP) FE_DEC_ROW(DP, F16, FE_DTYPE_F16) FE_DEC_ROW(DP, BF16, FE_DTYPE_BF16)
// Kernels by tile dim. rows and replay: the second takes operands whose rows all allow 16-byte loads. wide: of four
// waves, and of eight where their registers allow it.
struct DecKernels {
  int dp, dtype;
  const void* rows[2];
  const void* wide[2];
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
    const void* fns[7] = {e.rows[1], e.wide[0], e.wide[1], e.join, e.replay[1], e.rows[0], e.replay[0]};
    const char* names[7] = {"decode_rows", "decode_wide4", "decode_wide8", "decode_join", "decode_replay", "decode_rows_elements", "decode_replay_elements"};
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

// 16-byte loads of rows: unit channel stride, channels in whole 16-byte chunks, every row on a 16-byte boundary.
bool vec_ok(const void* p, const long long (&st)[4], int64_t B, int64_t H, int64_t N, int64_t D) {
  return D % 8 == 0 && st[3] == 1 && (uintptr_t)p % 16 == 0 && (B <= 1 || st[0] % 8 == 0) && (H <= 1 || st[1] % 8 == 0) &&
         (N <= 1 || st[2] % 8 == 0);
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
  if (C > (1LL << 30) || Hq / Hkv > 32767 || B > (1LL << 30) || Hkv > (1LL << 30) || B * Hkv > (1LL << 24) ||
      B * Hkv * ((C + T + 127) / 128) > 0x7fffffffLL || B * Hkv * (((Hq / Hkv) * T + 31) / 32) > 0x7fffffLL) {
    set_error(w + ": sizes exceed the supported range");
    return FE_ERR_UNSUPPORTED;
  }
  return FE_OK;
}

int dec_strides(const char* who, const int64_t* const* in, long long (*out[])[4], int count) {
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
      (*out[i])[j] = in[i][j];
    }
  }
  return FE_OK;
}

// How an attention launch is laid out; the same for the workspace's size and the call, whatever the layout of rows.
struct DecPlan {
  bool wide;
  int waves, RB, RW, nb;       // waves of a wide block; segments of a head, 32-row tiles of one, blocks
  long long slots;
  size_t o, ml, seg, logits, bytes;   // offsets
};
DecPlan dec_plan(int64_t BH, int64_t R, int64_t C, int64_t T, int64_t DP, bool vec, bool weights) {
  DecPlan p = {};
  const int64_t RT = (R + 31) / 32;
  p.wide = vec && RT > 1;
  if (p.wide) {
    p.waves = DP > 128 || RT <= 4 ? 4 : 8;
    p.RB = (int)((RT + p.waves - 1) / p.waves);
    p.RW = (int)((RT + p.RB - 1) / p.RB);
  } else {
    p.RB = (int)RT;
    p.RW = 1;
  }
  // As many blocks as the card holds at once, of at least a tile a wave.
  const int64_t KT = p.wide ? 64 : 32, tiles = BH * p.RB * ((C + KT - 1) / KT + (T + KT - 1) / KT);
  const int64_t resident = p.wide ? (p.waves == 8 || DP > 128 ? 256 : 512) : (DP > 128 ? 256 : 512);
  p.nb = (int)std::max<int64_t>(1, std::min(resident, p.wide ? tiles : (tiles + 3) / 4));
  p.slots = p.nb + BH * p.RB;
  auto area = [&](size_t elems) {
    const size_t at = p.bytes;
    p.bytes += (elems * 4 + 255) / 256 * 256;
    return at;
  };
  p.o = area((size_t)p.slots * p.RW * 32 * DP);
  p.ml = area((size_t)p.slots * p.RW * 64);
  p.seg = area((size_t)BH * p.RB * 2);
  p.logits = p.bytes;
  if (weights && R <= kDecLogitRows) area((size_t)BH * ((C + 31) / 32 + (T + 31) / 32) * R * 32);
  return p;
}

int dec_launch(const char* who, const void* fn, dim3 grid, dim3 block, DecArgs& a, hipStream_t stream) {
  void* args[] = {&a};
  hipError_t err = hipLaunchKernel(fn, grid, block, args, 0, stream);
  if (err != hipSuccess) {
    set_error(std::string(who) + ": launch: " + hipGetErrorString(err));
    return FE_ERR_HIP;
  }
  return FE_OK;
}

int dec_replay(const char* who, const DecKernels& kn, int vec, DecArgs& a, hipStream_t stream) {
  // as many blocks as the card holds at once, of at least a tile a wave
  const long long tiles = (long long)a.BH * ((a.C + 31) / 32 + (a.A + 31) / 32);
  a.nb = (int)std::max<long long>(1, std::min<long long>(kn.dp > 128 ? 512 : 768, (tiles + 3) / 4));
  return dec_launch(who, kn.replay[vec], dim3((unsigned)a.nb), dim3(256), a, stream);
}

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" size_t fe_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t C, int64_t D, int weights) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || T < 1 || C < 1 || D < 1 || D > 256 || T > kDecMaxTokens || B > (1LL << 24) ||
      Hkv > (1LL << 24) || Hq > (1LL << 24) || C > (1LL << 30) || B * Hkv > (1LL << 24) ||
      B * Hkv * ((Hq / Hkv * T + 31) / 32) > 0x7fffffLL)
    return 0;
  const int64_t dp = dec_kernels(D, 0).dp;
  return std::max(dec_plan(B * Hkv, Hq / Hkv * T, C, T, dp, false, weights != 0).bytes,
                  dec_plan(B * Hkv, Hq / Hkv * T, C, T, dp, true, weights != 0).bytes);
}

// The signs and zeros of Q that let a launch use a positive scale: a negative one runs as |scale| on -Q, a zero one
// as 1 on zeros (masked logits, -inf, times a zero scale would be NaN).
static void dec_scale(DecArgs& a, float scale, float decay) {
  a.qand = scale == 0.f ? 0u : ~0u;
  a.qxor = scale < 0.f ? 0x80008000u : 0u;
  a.scale_log2 = scale == 0.f ? 1.f : (float)(fabs((double)scale) * 1.4426950408889634);
  a.decay_log2 = (float)((double)decay * 1.4426950408889634);
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
  DecArgs a = {};
  const int64_t* in[5] = {q_strides, k_strides, v_strides, k_cache_strides, v_cache_strides};
  long long(*st[5])[4] = {&a.qs, &a.ks, &a.vs, &a.kcs, &a.vcs};
  if (int rc = dec_strides(who, in, st, 5)) return rc;
  const DecKernels& kn = dec_kernels(D, dtype);
  const size_t need = fe_decode_workspace_bytes(B, Hq, Hkv, T, C, D, importance != nullptr);
  if (!workspace || workspace_bytes < need) {
    set_error(std::string(who) + ": workspace too small; need " + std::to_string(need) + " bytes");
    return FE_ERR_WORKSPACE;
  }
  a.q = (const u16*)q;
  a.k = (const u16*)k;
  a.v = (const u16*)v;
  a.kc = (const u16*)k_cache;
  a.vc = (const u16*)v_cache;
  a.length = length;
  a.tree = tree;
  a.tree_stride = tree_batch_stride;
  a.out = (u16*)out;
  a.lse = lse;
  a.lse_in = lse;
  a.T = (int)T;
  a.A = (int)T;
  a.C = (int)C;
  a.D = (int)D;
  a.G = (int)(Hq / Hkv);
  a.Hkv = (int)Hkv;
  a.BH = (int)(B * Hkv);
  a.R = a.G * a.T;
  dec_scale(a, scale, recency_decay);
  const int vec = vec_ok(q, a.qs, B, Hq, T, D) && vec_ok(k, a.ks, B, Hkv, T, D) && vec_ok(v, a.vs, B, Hkv, T, D) &&
                  vec_ok(k_cache, a.kcs, B, Hkv, C, D) && vec_ok(v_cache, a.vcs, B, Hkv, C, D);
  const DecPlan p = dec_plan(a.BH, a.R, C, T, kn.dp, vec, importance != nullptr);
  const bool logits = importance && a.R <= kDecLogitRows;
  a.RB = p.RB;
  a.RW = p.RW;
  a.nb = p.nb;
  a.max_tiles = (int)((C + 31) / 32 + (T + 31) / 32);
  a.part_o = (float*)((char*)workspace + p.o);
  a.part_ml = (float*)((char*)workspace + p.ml);
  a.seg = (int*)((char*)workspace + p.seg);
  a.logits = logits ? (float*)((char*)workspace + p.logits) : nullptr;
  a.imp = importance;
  a.imp_stride = importance_stride;
  a.norm = value_norm;
  a.norm_stride = value_norm_stride;
  a.imp_out = importance_out;
  a.impo_stride = importance_out_stride;
  a.new_imp = new_importance;
  hipStream_t stream = (hipStream_t)hip_stream;
  if (p.wide) {
    if (int rc = dec_launch(who, kn.wide[p.waves == 8], dim3((unsigned)p.nb), dim3(64 * p.waves), a, stream)) return rc;
  } else {
    if (int rc = dec_launch(who, kn.rows[vec], dim3((unsigned)p.nb), dim3(256), a, stream)) return rc;
  }
  // eight groups on a row where it has many splits, else a group a row
  const long long rows = (long long)a.BH * a.R;
  a.join_split = p.nb >= 8 * a.BH * a.RB ? 8 : 1;
  a.join_blocks = (int)((rows * a.join_split + 7) / 8);
  const long long blocks = a.join_blocks + (logits ? (long long)a.BH * ((a.max_tiles + 7) / 8) : 0);
  if (int rc = dec_launch(who, kn.join, dim3((unsigned)blocks), dim3(256), a, stream)) return rc;
  if (logits) return FE_OK;
  if (!importance) return FE_OK;
  return dec_replay(who, kn, vec, a, stream);
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
  DecArgs a = {};
  const int64_t* in[4] = {q_strides, k_strides, v_strides, k_cache_strides};
  long long(*st[4])[4] = {&a.qs, &a.ks, &a.vs, &a.kcs};
  if (int rc = dec_strides(who, in, st, 4)) return rc;
  const DecKernels& kn = dec_kernels(D, dtype);
  a.q = (const u16*)q;
  a.k = (const u16*)k;
  a.v = (const u16*)v;
  a.kc = (const u16*)k_cache;
  a.length = length;
  a.lse_in = lse;
  a.path = path;
  a.T = (int)T;
  a.A = (int)A;
  a.C = (int)C;
  a.D = (int)D;
  a.G = (int)(Hq / Hkv);
  a.Hkv = (int)Hkv;
  a.BH = (int)(B * Hkv);
  dec_scale(a, scale, recency_decay);
  const int vec = vec_ok(q, a.qs, B, Hq, T, D) && vec_ok(k, a.ks, B, Hkv, T, D) && vec_ok(k_cache, a.kcs, B, Hkv, C, D);
  a.imp = importance;
  a.imp_stride = importance_stride;
  a.norm = value_norm;
  a.norm_stride = value_norm_stride;
  a.imp_out = importance_out;
  a.impo_stride = importance_out_stride;
  a.new_imp = new_importance;
  return dec_replay(who, kn, vec, a, (hipStream_t)hip_stream);
}
