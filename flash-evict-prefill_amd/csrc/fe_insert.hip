// Insertion of new tokens into a bounded KV cache, and the eviction of the rows of least accumulated attention
// weight, in place, for gfx950.
//
// For batch row b and KV head j: candidates are the n = length[b, j] cache rows at slots 0 .. n-1 and the A new rows
// (all T, or the nodes of path[b]), as if appended at slots n .. n+A-1 with positions seen .. seen+A-1. Of these
// F = min(n + A, budget) are kept: the newest `recent` ones (position >= seen + A - recent) first, then by importance
// (NaN above every number, -0 equal to +0), equal ones by slot. A kept candidate below F stays in its slot; the i-th
// one at or past F goes to the i-th slot below F that was vacated. So an insertion moves as many rows as it evicts,
// wherever they lie, and no row is both read and written: sources are new rows or slots at or past F, targets are
// vacated slots below F.
//
// One 1024-thread workgroup per (b, j): a radix select of the threshold over order keys, one ordered pass that lists
// the vacated slots and the rows that move, then a row per wave (half a wave on K, half on V).
#include <math.h>
#include <algorithm>
#include <string>

#include "fe_attn.h"
#include "fe_internal.h"
#include "fe_radix.h"
#include "../../include/flash_evict.h"

namespace fe {

struct InsArgs {
  const u16* k;
  const u16* v;
  u16* kc;
  u16* vc;
  float* imp;              // [B * Hkv] rows of imp_stride
  int* pos;
  float* norm;             // or null
  int* length;
  int* seen;
  const float* new_imp;    // [B * Hkv, A], or null: 0
  const int* path;         // [B, A], or null: all T
  int* lists;              // [B * Hkv][2][E]: vacated slots, moving candidates
  long long ks[4], vs[4], kcs[4], vcs[4];
  long long imp_stride, pos_stride, norm_stride;
  int T, A, C, D, Hkv, budget, recent, E;
  int bf16, kvec, vvec, kcvec, vcvec;
};

// Order key of a candidate: protected ones above NaN, NaN above every number.
__device__ __forceinline__ u32 ins_key(float w, bool held) { return held ? 0xffffffffu : min(order_key(w), 0xfffffffeu); }

// Copies row `src` of one operand to slot `dst` by 32 lanes (l32); returns the lane's sum of absolute values.
template <bool BF>
__device__ __forceinline__ float ins_row(const u16* from, long long fcs, int fvec, u16* to, long long tcs, int tvec, int D,
                                         int l32) {
  float sum = 0.f;
  for (int d = 8 * l32; d < D; d += 256) {
    const u32x4 x = load8(from, fcs, d, D, fvec);
    if (tvec) {
      *(u32x4*)(to + d) = x;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d + e < D) to[(long long)(d + e) * tcs] = (u16)(x[e >> 1] >> (16 * (e & 1)));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const u16 h = (u16)(x[e >> 1] >> (16 * (e & 1)));
      sum += fabsf(BF ? BF16::to_f32(h) : F16::to_f32(h));
    }
  }
  return sum;
}

__global__ __launch_bounds__(1024) void insert_kernel(const InsArgs a) {
  __shared__ u32 hist[2 * 2048];
  __shared__ __attribute__((aligned(16))) int tmp[2 * kSelWaves];
  __shared__ SelShared sh;
  __shared__ int s_len;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5, wv = tid >> 6;
  const int bh = (int)blockIdx.x, b = bh / a.Hkv, hkv = bh - b * a.Hkv;
  const int n = min(max(a.length[bh], 0), a.C);
  const int seen = a.seen[bh];
  const int* path = a.path ? a.path + (long long)b * a.A : nullptr;
  if (path) {
    // leading nodes that name one of the T tokens
    if (tid == 0) s_len = a.A;
    __syncthreads();
    for (int i = tid; i < a.A; i += 1024)
      if (path[i] < 0 || path[i] >= a.T) atomicMin(&s_len, i);
    __syncthreads();
  }
  const int na = path ? s_len : a.A;
  const int M = n + na, F = min(M, a.budget);
  const long long held = (long long)seen + na - a.recent;   // first protected position
  float* imp = a.imp + bh * a.imp_stride;
  int* pos = a.pos + bh * a.pos_stride;
  const float* fresh = a.new_imp ? a.new_imp + (long long)bh * a.A : nullptr;
  int* holes = a.lists + (long long)bh * 2 * a.E;
  int* movers = holes + a.E;

  auto get = [&](int i) -> u32 {
    if (i < n) return ins_key(imp[i], pos[i] >= held);
    return ins_key(fresh ? fresh[i - n] : 0.f, (long long)seen + (i - n) >= held);
  };
  int moves = 0;
  u32 thr = 0;
  int need = 0, eq = 0;
  if (M > F) {
    radix_select(get, M, F, 0u, 0xffffffffu, hist, tmp, &sh, thr, need, eq);
    int eq_before = 0, hole_before = 0, move_before = 0;
    for (int base = 0; base < M; base += 1024) {
      const int i = base + tid;
      const u32 key = i < M ? get(i) : 0u;
      bool kept = i < M && key > thr;
      if (need < eq) {
        int total;
        const int rank = eq_before + block_exclusive_scan(i < M && key == thr ? 1 : 0, tmp, total);
        eq_before += total;
        kept = kept || (i < M && key == thr && rank < need);
      } else {
        kept = kept || (i < M && key == thr);
      }
      const int hole = i < F && !kept, mover = i >= F && kept;
      int total;
      const int at = block_exclusive_scan(hole | (mover << 16), tmp, total);
      if (hole) holes[hole_before + (at & 0xffff)] = i;
      if (mover) movers[move_before + (at >> 16)] = i;
      hole_before += total & 0xffff;
      move_before += total >> 16;
    }
    moves = move_before;
  }
  __syncthreads();

  // the new rows that stay where they were appended, then the rows that move
  const u16* kn = a.k + b * a.ks[0] + hkv * a.ks[1];
  const u16* vn = a.v + b * a.vs[0] + hkv * a.vs[1];
  u16* kc = a.kc + b * a.kcs[0] + hkv * a.kcs[1];
  u16* vc = a.vc + b * a.vcs[0] + hkv * a.vcs[1];
  const int appended = max(F - n, 0);
  for (int j = wv; j < appended + moves; j += kSelWaves) {
    int src, dst;
    if (j < appended) {
      src = dst = n + j;
    } else {
      src = movers[j - appended];
      dst = holes[j - appended];
    }
    if (j < appended && M > F) {
      // a new row below F that was not kept: its slot is among the vacated ones
      const u32 key = get(src);
      bool kept = key > thr;
      if (key == thr) {
        kept = need == eq;
        if (!kept) {
          kept = true;
          for (int i = 0; i < moves; ++i) kept = kept && holes[i] != src;
        }
      }
      if (!kept) continue;
    }
    const bool is_new = src >= n;
    const int row = is_new ? (path ? path[src - n] : src - n) : src;
    float s;
    if (hh == 0) {
      const u16* from = is_new ? kn + (long long)row * a.ks[2] : kc + (long long)row * a.kcs[2];
      s = ins_row<true>(from, is_new ? a.ks[3] : a.kcs[3], is_new ? a.kvec : a.kcvec, kc + (long long)dst * a.kcs[2], a.kcs[3],
                        a.kcvec, a.D, l32);
    } else {
      const u16* from = is_new ? vn + (long long)row * a.vs[2] : vc + (long long)row * a.vcs[2];
      u16* to = vc + (long long)dst * a.vcs[2];
      const long long fcs = is_new ? a.vs[3] : a.vcs[3];
      const int fv = is_new ? a.vvec : a.vcvec;
      s = a.bf16 ? ins_row<true>(from, fcs, fv, to, a.vcs[3], a.vcvec, a.D, l32)
                 : ins_row<false>(from, fcs, fv, to, a.vcs[3], a.vcvec, a.D, l32);
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) s += __shfl_xor(s, d);
    if (lane == 32) {
      if (a.norm) {
        float* norm = a.norm + bh * a.norm_stride;
        norm[dst] = is_new ? s : norm[src];
      }
      imp[dst] = is_new ? (fresh ? fresh[src - n] : 0.f) : imp[src];
      pos[dst] = is_new ? seen + (src - n) : pos[src];
    }
  }
  if (tid == 0) {
    a.length[bh] = F;
    a.seen[bh] = seen + na;
  }
}

void append_insert_resources(std::string& out) {
  hipFuncAttributes attr;
  if (hipFuncGetAttributes(&attr, (const void*)insert_kernel) != hipSuccess) return;
  char buf[512];
  snprintf(buf, sizeof(buf),
           "{\"kernel\":\"insert_kernel\",\"registers_per_thread\":%d,\"lds_static_bytes\":%zu,"
           "\"lds_dynamic_bytes\":0,\"scratch_bytes_per_thread\":%zu,\"max_threads_per_block\":%d},",
           attr.numRegs, (size_t)attr.sharedSizeBytes, (size_t)attr.localSizeBytes, attr.maxThreadsPerBlock);
  out += buf;
}

namespace {
// Rows that an insertion can move: they come from past the budget and go below it.
int64_t ins_list(int64_t C, int64_t A, int64_t budget) { return std::max<int64_t>(0, std::min(C + A - budget, budget)); }
}  // namespace
}  // namespace fe

using namespace fe;

extern "C" size_t fe_insert_workspace_bytes(int64_t B, int64_t Hkv, int64_t A, int64_t C, int64_t budget) {
  if (B < 1 || Hkv < 1 || A < 0 || C < 1 || budget < 1 || budget > C || B > (1LL << 24) || Hkv > (1LL << 24) || A > (1LL << 29) ||
      C > (1LL << 30) || B * Hkv > (1LL << 24))
    return 0;
  return (size_t)(B * Hkv * 2 * ins_list(C, A, budget)) * sizeof(int);
}

extern "C" int fe_insert_tokens(const void* k, const void* v, void* k_cache, void* v_cache, float* importance,
                                int64_t importance_stride, int32_t* position, int64_t position_stride, float* value_norm,
                                int64_t value_norm_stride, int32_t* length, int32_t* seen, const float* new_importance,
                                const int32_t* path, int64_t B, int64_t Hkv, int64_t T, int64_t A, int64_t C, int64_t D,
                                int64_t budget, int64_t recent, const int64_t* k_strides, const int64_t* v_strides,
                                const int64_t* k_cache_strides, const int64_t* v_cache_strides, int dtype, void* workspace,
                                size_t workspace_bytes, void* hip_stream) {
  static const char* who = "fe_insert_tokens";
  clear_error();
  if (B < 1 || Hkv < 1 || T < 0 || A < 0 || A > T || (!path && A != T) || C < 1 || D < 1 || D > 256 || budget < 1 || budget > C ||
      recent < 0 || recent > budget) {
    set_error(std::string(who) + ": invalid shape, budget or recent");
    return FE_ERR_INVALID;
  }
  if (dtype != FE_DTYPE_F16 && dtype != FE_DTYPE_BF16) {
    set_error(std::string(who) + ": dtype must be fp16 or bf16");
    return FE_ERR_INVALID;
  }
  if (C > (1LL << 30) || T > (1LL << 29) || B > (1LL << 24) || Hkv > (1LL << 24) || B * Hkv > (1LL << 24)) {
    set_error(std::string(who) + ": sizes exceed the supported range");
    return FE_ERR_UNSUPPORTED;
  }
  if ((T && (!k || !v)) || !k_cache || !v_cache || !importance || !position || !length || !seen) {
    set_error(std::string(who) + ": null pointer argument");
    return FE_ERR_INVALID;
  }
  if (importance_stride < C || position_stride < C || (value_norm && value_norm_stride < C)) {
    set_error(std::string(who) + ": invalid row stride");
    return FE_ERR_INVALID;
  }
  const int64_t* in[4] = {k_strides, v_strides, k_cache_strides, v_cache_strides};
  InsArgs a = {};
  long long(*st[4])[4] = {&a.ks, &a.vs, &a.kcs, &a.vcs};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      if (!in[i] || in[i][j] < 0) {
        set_error(std::string(who) + ": null or negative strides");
        return FE_ERR_INVALID;
      }
      (*st[i])[j] = in[i][j];
    }
  const size_t need = fe_insert_workspace_bytes(B, Hkv, A, C, budget);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error(std::string(who) + ": workspace too small; need " + std::to_string(need) + " bytes");
    return FE_ERR_WORKSPACE;
  }
  auto vec = [&](const void* p, const long long(&s)[4], int64_t N) {
    return D % 8 == 0 && s[3] == 1 && (uintptr_t)p % 16 == 0 && (B <= 1 || s[0] % 8 == 0) && (Hkv <= 1 || s[1] % 8 == 0) &&
           (N <= 1 || s[2] % 8 == 0);
  };
  a.k = (const u16*)k;
  a.v = (const u16*)v;
  a.kc = (u16*)k_cache;
  a.vc = (u16*)v_cache;
  a.imp = importance;
  a.imp_stride = importance_stride;
  a.pos = position;
  a.pos_stride = position_stride;
  a.norm = value_norm;
  a.norm_stride = value_norm_stride;
  a.length = length;
  a.seen = seen;
  a.new_imp = new_importance;
  a.path = path;
  a.lists = (int*)workspace;
  a.T = (int)T;
  a.A = (int)A;
  a.C = (int)C;
  a.D = (int)D;
  a.Hkv = (int)Hkv;
  a.budget = (int)budget;
  a.recent = (int)recent;
  a.E = (int)ins_list(C, A, budget);
  a.bf16 = dtype == FE_DTYPE_BF16;
  a.kvec = vec(k, a.ks, T);
  a.vvec = vec(v, a.vs, T);
  a.kcvec = vec(k_cache, a.kcs, C);
  a.vcvec = vec(v_cache, a.vcs, C);
  hipLaunchKernelGGL(insert_kernel, dim3((unsigned)(B * Hkv)), dim3(1024), 0, (hipStream_t)hip_stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) {
    set_error(std::string(who) + ": launch: " + hipGetErrorString(err));
    return FE_ERR_HIP;
  }
  return FE_OK;
}
