// Selection by order keys within a workgroup: the order-preserving map of floats, prefix sums over waves and
// workgroups, and the radix select of the K-th largest key.
#pragma once

#include "fe_common.h"

namespace fe {

__device__ __forceinline__ u32 order_key(float f) {
  u32 u = __float_as_uint(f);
  if (f != f) return 0xffffffffu;  // NaN: above every number (torch.topk convention)
  if (u == 0x80000000u) u = 0u;    // -0.0 ties with +0.0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;                  // threads of a selection workgroup (one row)
constexpr int kSelWaves = kSelThreads / 64;

// The selection kernels synchronise through LDS with lds_barrier() (fe_common.h):
// __syncthreads() also waits for every outstanding global load and store of the wave, which
// would stall the row's streaming loads (and the mask stores) at each prefix sum. A full
// barrier is used only where global memory written by one thread is then read or
// overwritten by another.

// Inclusive prefix sum over the 64 lanes of a wave with DPP moves: shifts by 1, 2, 4 and 8
// lanes inside each 16-lane row, then the last lane of row r added to row r+1 (row_bcast:15,
// rows 1 and 3) and lane 31 to rows 2 and 3 (row_bcast:31). Lanes without a source add 0.
__device__ __forceinline__ int wave_inclusive_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31
  return x;
}

// Inclusive running minimum / maximum over the 64 lanes of a wave, the same DPP pattern as
// wave_inclusive_scan (lanes without a source take the identity): lane 63 holds the wave's.
__device__ __forceinline__ u32 wave_inclusive_min(u32 x) {
  int v = (int)x;
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x111, 0xf, 0xf, false));
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x112, 0xf, 0xf, false));
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x114, 0xf, 0xf, false));
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x118, 0xf, 0xf, false));
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x142, 0xa, 0xf, false));
  v = min((u32)v, (u32)__builtin_amdgcn_update_dpp(-1, v, 0x143, 0xc, 0xf, false));
  return (u32)v;
}
__device__ __forceinline__ u32 wave_inclusive_max(u32 x) {
  int v = (int)x;
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max((u32)v, (u32)__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return (u32)v;
}

// Exclusive prefix sum over the threads of a selection workgroup; `total` receives the sum.
// tmp: kSelWaves ints, 16-byte aligned.
__device__ __forceinline__ int block_exclusive_scan(int v, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int x = wave_inclusive_scan(v);
  if (lane == 63) tmp[w] = x;
  lds_barrier();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSelWaves; ++i) {
    const int t = tmp[i];
    before += (i < w) ? t : 0;
    total += t;
  }
  lds_barrier();
  return before + x - v;
}

struct SelShared {
  u32 prefix;
  int kk;
  u32 eq;
};

// Radix select over n keys (key i = get(i)) for T = the K-th largest key (1 <= K <= n),
// need = how many keys equal to T are among the K largest, eq = how many keys equal T.
// Only keys in [lo, hi] are histogrammed; keys above hi are counted first. Returns false
// (T undetermined) when the K-th largest key lies outside [lo, hi]; the full range
// [0, 0xffffffff] always succeeds. The leading digits that lo and hi share are the same for
// every key in [lo, hi], so their passes are skipped.
//
// Three LDS-only barriers per pass: after the histogram (whose successor, in the other half
// of hist, is cleared meanwhile), after the per-wave sums of the bins each wave owns (every
// thread then finds the wave holding the K-th key from 16 sums), and after the digit, found
// by that wave alone, is published. hist: 2 x 2048 u32; tmp: 2 x kSelWaves ints.
template <typename Get>
__device__ __forceinline__ bool radix_select(Get get, int n, int K, u32 lo, u32 hi, u32* hist, int* tmp,
                                             SelShared* sh, u32& T, int& need, int& eq) {
  constexpr int ST = kSelThreads;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  u32 prefix = 0, pmask = 0, eq_total = 0;
  int kk = K;
  int first = 0;
  if ((lo >> 21) == (hi >> 21)) {
    first = 1;
    pmask = 0xffe00000u;
    if ((lo >> 10) == (hi >> 10)) {
      first = 2;
      pmask = 0xfffffc00u;
    }
    prefix = lo & pmask;
  }
  for (int i = tid; i < (first == 2 ? 1024 : 2048); i += ST) hist[(first & 1) * 2048 + i] = 0u;
  lds_barrier();
  for (int pass = first; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int nb = pass == 2 ? 1024 : 2048;
    u32* h = hist + (pass & 1) * 2048;
    if (pass < 2) {
      // the next pass's histogram: its last reader finished before this pass began
      u32* hn = hist + ((pass + 1) & 1) * 2048;
      for (int i = tid; i < (pass + 1 == 2 ? 1024 : 2048); i += ST) hn[i] = 0u;
    }
    int above = 0;
#pragma unroll 8
    for (int i = tid; i < n; i += ST) {
      const u32 key = get(i);
      if (pass == first) above += key > hi ? 1 : 0;
      if (key >= lo && key <= hi && (key & pmask) == prefix) atomicAdd(&h[(key >> shift) & (u32)(nb - 1)], 1u);
    }
    lds_barrier();
    // wave w owns bins [nb - (w+1)*bpw, nb - w*bpw), lane l the bpl of them below
    // nb - 1 - w*bpw - l*bpl: wave 0, lane 0 hold the highest digits
    const int bpw = nb / kSelWaves, bpl = bpw / 64;
    const int top = nb - 1 - w * bpw - lane * bpl;
    int lsum = 0;
    for (int e = 0; e < bpl; ++e) lsum += (int)h[top - e];
    const int incl = wave_inclusive_scan(lsum);
    const int wa = pass == first ? wave_inclusive_scan(above) : 0;
    if (lane == 63) {
      tmp[w] = incl;
      tmp[kSelWaves + w] = wa;
    }
    lds_barrier();
    int total = 0, n_above = 0, cw = -1, before = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
      total += tmp[i];
      n_above += pass == first ? tmp[kSelWaves + i] : 0;
    }
    if (pass == first) kk = K - n_above;
    if (pass == first && (kk < 1 || kk > total)) return false;   // uniform: block totals
    {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kSelWaves; ++i) {
        const int t = tmp[i];
        if (cw < 0 && c + t >= kk) {
          cw = i;
          before = c;
        }
        c += t;
      }
    }
    if (w == cw) {
      int c = before + incl - lsum;            // keys in the bins above this lane's
      if (c < kk && c + lsum >= kk) {
        for (int e = 0; e < bpl; ++e) {
          const int bin = top - e;
          const int hv = (int)h[bin];
          if (c < kk && c + hv >= kk) {
            sh->prefix = prefix | ((u32)bin << shift);
            sh->kk = kk - c;
            sh->eq = (u32)hv;
          }
          c += hv;
        }
      }
    }
    lds_barrier();
    prefix = sh->prefix;
    kk = sh->kk;
    eq_total = sh->eq;
    pmask |= (u32)(nb - 1) << shift;
  }
  T = prefix;
  need = kk;
  eq = (int)eq_total;
  return true;
}

}  // namespace fe
