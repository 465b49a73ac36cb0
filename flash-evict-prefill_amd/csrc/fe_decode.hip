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
//   decode_attn_kernel     a split of the keys for 32 query rows of a group (rows r = g * T + t): one pass with the
//                          running maximum and sum, S^T = K Q^T and O^T = V^T P^T on MFMA
//   decode_combine_kernel  joins the splits: out and lse
//   decode_replay_kernel   S = Q K^T again for the rows that stay, with lanes holding keys, so that a key's sum over
//                          the rows is in-lane: p = exp2(x log2e - bias), the bias holding lse and w
#include <math.h>
#include <algorithm>
#include <string>

#include "fe_attn.h"
#include "fe_internal.h"
#include "../../include/flash_evict.h"

namespace fe {

typedef __attribute__((address_space(3))) void* dec_lds_ptr;
typedef short dec_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) dec_s16x4 dec_lds_s16x4;

constexpr int kDecMaxTokens = 256;   // new tokens of a call

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
  float* part_o;           // [item][DP][32]
  float* part_ml;          // [item][2][32]: max (log2 units), sum
  long long qs[4], ks[4], vs[4], kcs[4], vcs[4];
  long long imp_stride, norm_stride, impo_stride, tree_stride;
  int T, C, D, G, Hkv, BH, A;
  int R, RB, S;            // rows of a group, 32-row blocks, key splits
  float scale_log2, decay_log2;
};

constexpr float kLn2 = 0.6931471805599453f;

// Rows of the (b, j) cache, within the tensor whatever the caller's length says.
__device__ __forceinline__ int dec_len(const DecArgs& a, int bh) { return min(max(a.length[bh], 0), a.C); }

// Orders a wave's own LDS writes and reads (the hardware keeps them in order; the compiler is told).
__device__ __forceinline__ void dec_wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// A wave's tile of 32 K rows in LDS: [16-channel pair c][32 keys][32 B], the two 16-byte chunks of a key swapped
// where key bit 3 is set; 32 V rows: [32-channel tile][32 keys][64 B]. Both as in the prefill kernels: the 16
// lanes of a fragment read's phase hit every bank once.
__device__ __forceinline__ int dec_k_at(int key, int chunk) {
  return (chunk >> 1) * 1024 + key * 32 + (((chunk & 1) ^ ((key >> 3) & 1)) << 4);
}
__device__ __forceinline__ int dec_v_at(int key, int chunk) { return (chunk >> 2) * 2048 + key * 64 + ((chunk & 3) << 4); }

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

template <typename E, int DP, int VEC>
__global__ __launch_bounds__(256) void decode_attn_kernel(const DecArgs a) {
  constexpr int NDC = DP / 16, NDT = DP / 32, CPR = DP / 8, TILE = 64 * DP;   // bytes of 32 rows
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][2 * TILE];
  __shared__ float sm[4][2][32];
  __shared__ float sp[4][32][33];        // probabilities of a tile with a value that is not finite
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int item = (int)blockIdx.x;
  const int bh = item % a.BH;
  item /= a.BH;
  const int sp_i = item % a.S, rb = item / a.S;
  const int b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  const int n = dec_len(a, bh);
  const int nc = (n + 31) / 32, nt = (a.T + 31) / 32, tiles = nc + nt;
  const int t_lo = (int)((long long)tiles * sp_i / a.S), t_hi = (int)((long long)tiles * (sp_i + 1) / a.S);

  const int r = rb * 32 + l32;           // this lane's query row
  const bool rv = r < a.R;
  const int g = rv ? r / a.T : 0, tq = rv ? r - g * a.T : 0;
  u32x4 qf[NDC];
  {
    const u16* qp = a.q + b * a.qs[0] + (hkv * a.G + g) * a.qs[1] + tq * a.qs[2];
#pragma unroll
    for (int c = 0; c < NDC; ++c) {
      qf[c] = rv ? dec_load8<VEC>(qp, a.qs[3], 2 * c + hh, a.D) : (u32x4){0u, 0u, 0u, 0u};
      if (!VEC) __builtin_amdgcn_sched_barrier(0);   // element loads: one chunk's addresses at a time
    }
  }
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = (f32x16){};
  float m = NEG_INF, l = 0.f, lr = 0.f;   // sums of the probabilities, and of these as rounded for the product

  unsigned char* kt = lds[wv];
  unsigned char* vt = lds[wv] + TILE;
  for (int t = t_lo + wv; t < t_hi; t += 4) {
    const bool tail = t >= nc;
    const int kb = tail ? (t - nc) * 32 : t * 32, rows = tail ? a.T : n;
    const u16* kp = tail ? a.k + b * a.ks[0] + hkv * a.ks[1] : a.kc + b * a.kcs[0] + hkv * a.kcs[1];
    const u16* vp = tail ? a.v + b * a.vs[0] + hkv * a.vs[1] : a.vc + b * a.vcs[0] + hkv * a.vcs[1];
    const long long krs = tail ? a.ks[2] : a.kcs[2], kcs = tail ? a.ks[3] : a.kcs[3];
    const long long vrs = tail ? a.vs[2] : a.vcs[2], vcs = tail ? a.vs[3] : a.vcs[3];
    // keys of the tail whose value has an infinity or a NaN: 0 * inf would reach the rows that do not see
    // them, so their values are taken out of the product and added to the rows that do
    u32 odd = 0;
    constexpr int U = VEC ? NDC : 1;        // chunks in flight
#pragma unroll 1
    for (int i0 = 0; i0 < NDC; i0 += U) {
      u32x4 kx[U], vx[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int e = (i0 + i) * 64 + lane, row = kb + e / CPR, ch = e % CPR;
        kx[i] = row < rows ? dec_load8<VEC>(kp + (long long)row * krs, kcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
        vx[i] = row < rows ? dec_load8<VEC>(vp + (long long)row * vrs, vcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int e = (i0 + i) * 64 + lane, key = e / CPR, ch = e % CPR;
        if (tail)
          for (unsigned long long bl = __ballot(dec_nonfinite<E>(vx[i])); bl; bl &= bl - 1)
            odd |= 1u << (((i0 + i) * 64 + __ffsll(bl) - 1) / CPR);
        *(u32x4*)(kt + dec_k_at(key, ch)) = kx[i];
        *(u32x4*)(vt + dec_v_at(key, ch)) = vx[i];
      }
    }
    if (odd) {
      dec_wave_order();
      for (int e = lane; e < 32 * CPR; e += 64)
        if ((odd >> (e / CPR)) & 1u) *(u32x4*)(vt + dec_v_at(e / CPR, e % CPR)) = (u32x4){0u, 0u, 0u, 0u};
    }
    dec_wave_order();
    // S^T: lanes hold queries; register i holds key kb + 8 (i / 4) + 4 hh + i % 4
    f32x16 x;
#pragma unroll
    for (int c = 0; c < NDC; ++c) {
      const u32x4 kf = *(const u32x4*)(kt + c * 1024 + l32 * 32 + ((hh ^ ((l32 >> 3) & 1)) << 4));
      x = c == 0 ? E::mfma(kf, qf[0], (f32x16){}) : E::mfma(kf, qf[c], x);
    }
    u32 vis = 0;                            // bit i: register i's key is visible to this lane's query
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = kb + 8 * (i >> 2) + 4 * hh + (i & 3);
      bool see = key < rows;
      if (tail) {
        if (!a.tree) see = key <= tq;
        else see = see && a.tree[b * a.tree_stride + tq * a.T + (see ? key : 0)] != 0;
      }
      see = see && rv;
      vis |= (see ? 1u : 0u) << i;
      x[i] = see ? x[i] * a.scale_log2 : NEG_INF;
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < 16; ++i) mn = fmaxf(mn, x[i]);
    mn = half_swap_max(mn);
    const float ref = mn == NEG_INF ? 0.f : mn;
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
    // O^T += V^T P^T over the tile's two 16-key groups; the transposing reads give a lane eight keys of one
    // channel in the accumulators' key order
    const int tr = lane & 15, tg = lane >> 4;
    const int voff = (4 * hh + (tr >> 2)) * 64 + 32 * (tg & 1) + 8 * (tr & 3);
#pragma unroll
    for (int c4 = 0; c4 < 2; ++c4) {
      const u32x4 pf = {pw[4 * c4], pw[4 * c4 + 1], pw[4 * c4 + 2], pw[4 * c4 + 3]};
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        unsigned char* p = vt + dt * 2048 + c4 * 1024 + voff;
        const u32x2 ux = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)p));
        const u32x2 uy = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((dec_lds_s16x4*)(dec_lds_ptr)(p + 512)));
        o[dt] = E::mfma((u32x4){ux[0], ux[1], uy[0], uy[1]}, pf, o[dt]);
      }
    }
    if (odd) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sp[wv][8 * (i >> 2) + 4 * hh + (i & 3)][l32] = (vis >> i) & 1u ? x[i] : -1.f;
      dec_wave_order();
      const u16* vb = a.v + b * a.vs[0] + hkv * a.vs[1];
      for (u32 left = odd; left; left &= left - 1) {
        const int key = __ffs((int)left) - 1;
        const float p = sp[wv][key][l32];
        float* row = (float*)kt;            // the value's channels; K is done with
        for (int ch = lane; ch < DP; ch += 64) row[ch] = ch < a.D ? E::to_f32(vp[(long long)(kb + key) * vrs + ch * vcs]) : 0.f;
        dec_wave_order();
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = row[32 * dt + 8 * (i >> 2) + 4 * hh + (i & 3)];
            if (p >= 0.f) o[dt][i] += p * x;
          }
        dec_wave_order();
      }
    }
    dec_wave_order();                       // the next tile's stores follow this one's reads
  }

  // join the four waves: [channel][32 rows] of each in its own tiles' LDS
  if (hh == 0) {
    sm[wv][0][l32] = m;
    sm[wv][1][l32] = l;
  }
  __shared__ float sl[4][32];
  if (hh == 0) sl[wv][l32] = lr;
  float* mine = (float*)lds[wv];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) mine[(32 * dt + 8 * (i >> 2) + 4 * hh + (i & 3)) * 32 + l32] = o[dt][i];
  __syncthreads();
  float mx = fmaxf(fmaxf(sm[0][0][l32], sm[1][0][l32]), fmaxf(sm[2][0][l32], sm[3][0][l32]));
  const float ref = mx == NEG_INF ? 0.f : mx;
  float w[4], ltot = 0.f, lrtot = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = fast_exp2(sm[i][0][l32] - ref);
    ltot += sm[i][1][l32] * w[i];
    lrtot += sl[i][l32] * w[i];
  }
  // partials are normalised by the sum of the rounded probabilities, and weighted by the exact one: so a row that
  // one key dominates returns that key's value whatever the split
  const float inv = lrtot > 0.f ? 1.f / lrtot : (lrtot == 0.f ? 0.f : lrtot);
  const long long it = ((long long)bh * a.RB + rb) * a.S + sp_i;
  if (threadIdx.x < 32) {
    a.part_ml[it * 64 + l32] = mx;
    a.part_ml[it * 64 + 32 + l32] = ltot;
  }
  float* po = a.part_o + it * (DP * 32);
  for (int ch = threadIdx.x >> 5; ch < DP; ch += 8) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += w[i] * ((float*)lds[i])[ch * 32 + l32];
    po[ch * 32 + l32] = s * inv;
  }
}

// One 32-row block of a (b, j): out = sum_s w_s O_s / sum w_s, w_s = l_s 2^(m_s - m).
template <typename E, int DP>
__global__ __launch_bounds__(256) void decode_combine_kernel(const DecArgs a) {
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ float tile[32][33];
  __shared__ float sm[8][32], sl[8][32];
  const int row = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int blk = (int)blockIdx.x;          // bh * RB + rb
  const int bh = blk / a.RB, rb = blk - bh * a.RB, dt = (int)blockIdx.y;
  const int b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  const float* ml = a.part_ml + (long long)blk * a.S * 64;
  float m = NEG_INF;
  for (int s = part; s < a.S; s += 8) m = fmaxf(m, ml[s * 64 + row]);
  sm[part][row] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, sm[i][row]);
  const float ref = m == NEG_INF ? 0.f : m;
  float l = 0.f;
  for (int s = part; s < a.S; s += 8) l += ml[s * 64 + 32 + row] * fast_exp2(ml[s * 64 + row] - ref);
  sl[part][row] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) l += sl[i][row];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float* po = a.part_o + (long long)blk * a.S * (DP * 32) + dt * 32 * 32;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int ch = part + 8 * j;
    float acc = 0.f;
    for (int s = 0; s < a.S; ++s) {
      const float w = ml[s * 64 + 32 + row] * fast_exp2(ml[s * 64 + row] - ref);
      // a split that this row sees nothing of has a weight of 0 and values of 0
      acc += w * po[(long long)s * (DP * 32) + ch * 32 + row];
    }
    tile[row][ch] = acc * inv;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * 32; e += 256) {
    const int rr = e >> 5, ch = e & 31, r = rb * 32 + rr, d = dt * 32 + ch;
    if (r < a.R && d < a.D) {
      const int g = r / a.T, t = r - g * a.T;
      const u32 w = E::pack2(tile[rr][ch], 0.f);
      a.out[(((long long)b * a.Hkv * a.G + hkv * a.G + g) * a.T + t) * a.D + d] = (u16)w;
    }
  }
  if (dt == 0 && threadIdx.x < 32 && rb * 32 + row < a.R) {
    const int r = rb * 32 + row, g = r / a.T, t = r - g * a.T;
    a.lse[((long long)b * a.Hkv * a.G + hkv * a.G + g) * a.T + t] = l == 0.f ? NEG_INF : (m + fast_log2(l)) * kLn2;
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

template <typename E, int DP, int VEC>
__global__ __launch_bounds__(256) void decode_replay_kernel(const DecArgs a) {
  constexpr int NDC = DP / 16, CPR = DP / 8, TILE = 64 * DP;
  constexpr int CH = 256;                  // rows whose biases and places are in LDS at a time
  constexpr float POS_INF = __builtin_huge_valf();
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][TILE];
  __shared__ float bias[CH];
  __shared__ int place[CH];                // g * 65536 + node
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = (int)(blockIdx.x % (unsigned)a.BH), blk = (int)(blockIdx.x / (unsigned)a.BH);
  const int b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  const int n = dec_len(a, bh);
  const int nc = (n + 31) / 32, nt = (a.A + 31) / 32, tiles = nc + nt;
  if (blk * 4 >= tiles) return;
  const int na = dec_path_len(a, b), rows = a.G * na;
  const int t = blk * 4 + wv;
  const bool live = t < tiles, tail = t >= nc;
  const int kb = tail ? (t - nc) * 32 : t * 32;

  u32x4 kf[NDC];
  {
    const u16* kp = tail ? a.k + b * a.ks[0] + hkv * a.ks[1] : a.kc + b * a.kcs[0] + hkv * a.kcs[1];
    const long long krs = tail ? a.ks[2] : a.kcs[2], kcs = tail ? a.ks[3] : a.kcs[3];
    const int krows = !live ? 0 : (tail ? na : n);
    constexpr int U = VEC ? NDC : 1;
#pragma unroll 1
    for (int i0 = 0; i0 < NDC; i0 += U) {
      u32x4 kx[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int e = (i0 + i) * 64 + lane, key = kb + e / CPR, ch = e % CPR;
        const int row = tail && a.path && key < krows ? a.path[(long long)b * a.A + key] : key;   // new rows in the path's order
        kx[i] = key < krows ? dec_load8<VEC>(kp + (long long)row * krs, kcs, ch, a.D) : (u32x4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int e = (i0 + i) * 64 + lane;
        *(u32x4*)(lds[wv] + dec_k_at(e / CPR, e % CPR)) = kx[i];
      }
    }
    dec_wave_order();
#pragma unroll
    for (int c = 0; c < NDC; ++c) kf[c] = *(const u32x4*)(lds[wv] + c * 1024 + l32 * 32 + ((hh ^ ((l32 >> 3) & 1)) << 4));
  }

  float sum = 0.f;
  for (int r0 = 0; r0 < rows; r0 += CH) {
    __syncthreads();
    {
      const int r = r0 + (int)threadIdx.x;
      float bs = POS_INF;
      int pl = 0;
      if (r < rows) {
        const int g = r / na, i = r - g * na;
        const int node = a.path ? a.path[(long long)b * a.A + i] : i;
        const float z = a.lse_in[((long long)b * a.Hkv * a.G + hkv * a.G + g) * a.T + node];
        // nothing visible (lse = -inf): the row gives no weight
        bs = z == -POS_INF ? POS_INF : z * (1.f / kLn2) + a.decay_log2 * (float)(na - 1 - i);
        pl = (g << 16) | node;
      }
      bias[threadIdx.x] = bs;
      place[threadIdx.x] = pl;
    }
    __syncthreads();
    const int rend = min(CH, rows - r0);
    for (int rt = 0; rt < rend; rt += 32) {
      // lanes hold keys; register i holds row rt + 8 (i / 4) + 4 hh + i % 4
      const int pl = place[rt + l32];
      const u16* qp = a.q + b * a.qs[0] + (hkv * a.G + (pl >> 16)) * a.qs[1] + (pl & 0xffff) * a.qs[2];
      f32x16 x;
#pragma unroll
      for (int c = 0; c < NDC; ++c) {
        const u32x4 qf = rt + l32 < rend ? dec_load8<VEC>(qp, a.qs[3], 2 * c + hh, a.D) : (u32x4){0u, 0u, 0u, 0u};
        x = c == 0 ? E::mfma(qf, kf[0], (f32x16){}) : E::mfma(qf, kf[c], x);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int rr = rt + 8 * (i >> 2) + 4 * hh + (i & 3);
        float p = fast_exp2(x[i] * a.scale_log2 - bias[rr]);
        // row i of the path sees new row u <= i
        if (rr >= rend || (tail && (r0 + rr) % na < kb + l32)) p = 0.f;
        sum += p;
      }
    }
  }
  sum = half_swap_sum(sum);
  if (!live || hh) return;
  const int key = kb + l32;
  if (!tail) {
    if (key < n) {
      const float old = a.imp[bh * a.imp_stride + key] * fast_exp2(-a.decay_log2 * (float)na);
      const float w = a.norm ? a.norm[bh * a.norm_stride + key] : 1.f;
      a.imp_out[bh * a.impo_stride + key] = old + w * sum;
    }
  } else if (key < a.A) {
    float w = 0.f;
    if (key < na) {
      w = 1.f;
      if (a.norm) {
        const int node = a.path ? a.path[(long long)b * a.A + key] : key;
        const u16* vp = a.v + b * a.vs[0] + hkv * a.vs[1] + node * a.vs[2];
        w = 0.f;
        for (int d = 0; d < a.D; ++d) w += fabsf(E::to_f32(vp[d * a.vs[3]]));
      }
    }
    a.new_imp[(long long)bh * a.A + key] = key < na ? w * sum : 0.f;
  }
}

#define FE_DEC_DIMS(X) X(64) X(96) X(128) X(192) X(256)
#define FE_DEC_ROW(DP, E, T)                                                                                            \
  {DP, T, {(const void*)decode_attn_kernel<E, DP, 0>, (const void*)decode_attn_kernel<E, DP, 1>},                       \
   (const void*)decode_combine_kernel<E, DP>,                                                                           \
   {(const void*)decode_replay_kernel<E, DP, 0>, (const void*)decode_replay_kernel<E, DP, 1>}},
#define FE_DEC_ROWS(DP) FE_DEC_ROW(DP, F16, FE_DTYPE_F16) FE_DEC_ROW(DP, BF16, FE_DTYPE_BF16)
// Kernels by tile dim; the second of a pair takes operands whose rows all allow 16-byte loads.
struct DecKernels {
  int dp, dtype;
  const void* attn[2];
  const void* combine;
  const void* replay[2];
};
const DecKernels kDecKernels[] = {FE_DEC_DIMS(FE_DEC_ROWS)};

const DecKernels& dec_kernels(int64_t D, int dtype) {
  for (const auto& e : kDecKernels)
    if (e.dp >= D && e.dtype == dtype) return e;
  return kDecKernels[0];
}

// Key splits of an attention launch: enough blocks to fill the CUs twice, each with at least four tiles of 32
// keys per wave.
int dec_splits(int64_t BH, int64_t RB, int64_t C, int64_t T) {
  const int64_t tiles = (C + 31) / 32 + (T + 31) / 32;
  int64_t s = (512 + BH * RB - 1) / (BH * RB);
  s = std::min<int64_t>(s, (tiles + 15) / 16);
  return (int)std::max<int64_t>(1, s);
}

void append_decode_resources(std::string& out) {
  for (const auto& e : kDecKernels) {
    const void* fns[5] = {e.attn[1], e.combine, e.replay[1], e.attn[0], e.replay[0]};
    const char* names[5] = {"decode_attn", "decode_combine", "decode_replay", "decode_attn_elements", "decode_replay_elements"};
    for (int i = 0; i < 5; ++i) {
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

size_t dec_ws_bytes(int64_t BH, int64_t R, int64_t C, int64_t T, int64_t DP) {
  const int64_t RB = (R + 31) / 32;
  return (size_t)(BH * RB * dec_splits(BH, RB, C, T)) * (size_t)(DP * 32 + 64) * sizeof(float);
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
  const long long tiles = (a.C + 31) / 32 + (a.A + 31) / 32, blocks = (tiles + 3) / 4 * a.BH;
  return dec_launch(who, kn.replay[vec], dim3((unsigned)blocks), dim3(256), a, stream);
}

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" size_t fe_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t C, int64_t D) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || T < 1 || C < 1 || D < 1 || D > 256 || T > kDecMaxTokens || B > (1LL << 24) ||
      Hkv > (1LL << 24) || Hq > (1LL << 24) || C > (1LL << 30) || B * Hkv > (1LL << 24) ||
      B * Hkv * ((Hq / Hkv * T + 31) / 32) > 0x7fffffLL)
    return 0;
  return dec_ws_bytes(B * Hkv, Hq / Hkv * T, C, T, dec_kernels(D, 0).dp);
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
  const size_t need = dec_ws_bytes(B * Hkv, Hq / Hkv * T, C, T, kn.dp);
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
  a.RB = (a.R + 31) / 32;
  a.S = dec_splits(a.BH, a.RB, C, T);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.decay_log2 = (float)((double)recency_decay * 1.4426950408889634);
  const int vec = vec_ok(q, a.qs, B, Hq, T, D) && vec_ok(k, a.ks, B, Hkv, T, D) && vec_ok(v, a.vs, B, Hkv, T, D) &&
                  vec_ok(k_cache, a.kcs, B, Hkv, C, D) && vec_ok(v_cache, a.vcs, B, Hkv, C, D);
  const long long items = (long long)a.BH * a.RB * a.S;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + items * kn.dp * 32;
  hipStream_t stream = (hipStream_t)hip_stream;
  if (int rc = dec_launch(who, kn.attn[vec], dim3((unsigned)items), dim3(256), a, stream)) return rc;
  if (int rc = dec_launch(who, kn.combine, dim3((unsigned)(a.BH * a.RB), (unsigned)(kn.dp / 32)), dim3(256), a, stream)) return rc;
  if (!importance) return FE_OK;
  a.imp = importance;
  a.imp_stride = importance_stride;
  a.norm = value_norm;
  a.norm_stride = value_norm_stride;
  a.imp_out = importance_out;
  a.impo_stride = importance_out_stride;
  a.new_imp = new_importance;
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
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.decay_log2 = (float)((double)recency_decay * 1.4426950408889634);
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
