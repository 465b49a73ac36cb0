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
//   insert_few_kernel    up to 256 new rows and 256 evicted ones, on caches of up to 32512 slots: one 1024-thread block a
//                        head. Order keys are staged in LDS; up to 32 victims are drawn one by one as the least key (of equal
//                        ones the highest slot), more are found by a radix select and an ordered pass
//   insert_list_kernel   otherwise: the same by a radix select over the head's rows in memory; leaves the list of moves
//   insert_move_kernel   carries it out, the whole card on it
#include <math.h>
#include <stddef.h>
#include <algorithm>
#include <string>
#include <type_traits>

#include "fe_attn.h"
#include "fe_internal.h"
#include "fe_radix.h"
#include "../../include/flash_evict.h"

namespace fe {

#define FE_GLOBAL __attribute__((address_space(1)))
typedef const FE_GLOBAL u16* InsIn;
typedef FE_GLOBAL u16* InsOut;

// New rows, and evicted ones, of insert_few_kernel: 40 to 250 rows into 8192 take it 32 us, the other two kernels 40.
constexpr int kInsFew = 256;
constexpr int kInsKeys = 32768;      // its candidates (128 KiB of LDS)
// Victims drawn one by one, 0.55 us each: 16 of 8192 rows 13.8 us, by selection 33.
constexpr int kInsDraw = 32;

struct InsArgs {
  InsIn k, v;
  InsOut kc, vc;
  FE_GLOBAL float* imp;    // [B * Hkv] rows of imp_stride
  FE_GLOBAL int* pos;
  FE_GLOBAL float* norm;   // or null
  FE_GLOBAL int* length;
  FE_GLOBAL int* seen;
  const FE_GLOBAL float* new_imp;    // [B * Hkv, A], or null: 0
  const FE_GLOBAL int* path;         // [B, A], or null: all T
  FE_GLOBAL int* lists;    // [B * Hkv][4 + 2 P]: pairs from the front, rows that stay from the back, n, seen; slots; sources
  long long kb, kh, kn, vb, vh, vn, kcb, kch, kcn, vcb, vch, vcn;   // strides of batch, head, row
  long long imp_stride, pos_stride, norm_stride;
  int T, A, C, D, Hkv, budget, recent, P, bf16;
  int pad;
  long long kd, vd, kcd, vcd;   // channel strides
};
static_assert(offsetof(InsArgs, kd) == 4 * 64, "argument window");

// The arguments, read at once and kept in registers, not one by one where they are used with a wait each time.
__device__ __forceinline__ InsArgs ins_hold(const InsArgs& arg) {
  InsArgs a = arg;
  typedef u32 u32x16 __attribute__((ext_vector_type(16), aligned(4)));
  typedef const __attribute__((address_space(4))) u32x16* args_ptr;
  const args_ptr p = (args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
  u32x16 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = p[i];
  asm volatile("" : "+s"(v[0]), "+s"(v[1]), "+s"(v[2]), "+s"(v[3]));
  u32 w[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    w[i] = v[i / 16][i % 16];
    asm volatile("" : "+s"(w[i]));
  }
  __builtin_memcpy(&a, w, 4 * 64);
  return a;
}

// Order keys: a drawn victim above everything, then protected candidates, NaN, numbers.
constexpr u32 kKeyDrawn = 0xffffffffu, kKeyHeld = 0xfffffffeu, kKeyNan = 0xfffffffdu;
__device__ __forceinline__ u32 ins_key(float w, bool held) { return held ? kKeyHeld : min(order_key(w), kKeyNan); }

// A head: its candidates and what they become.
struct InsHead {
  InsIn kn, vn;
  InsOut kc, vc;
  FE_GLOBAL float* imp;
  FE_GLOBAL int* pos;
  FE_GLOBAL float* norm;
  const FE_GLOBAL float* fresh;
  const FE_GLOBAL int* path;
  int n, seen;
};
__device__ __forceinline__ InsHead ins_head(const InsArgs& a, int b, int hkv, int n, int seen) {
  const long long bh = (long long)b * a.Hkv + hkv;
  InsHead h;
  h.kn = a.k + b * a.kb + hkv * a.kh;
  h.vn = a.v + b * a.vb + hkv * a.vh;
  h.kc = a.kc + b * a.kcb + hkv * a.kch;
  h.vc = a.vc + b * a.vcb + hkv * a.vch;
  h.imp = a.imp + bh * a.imp_stride;
  h.pos = a.pos + bh * a.pos_stride;
  h.norm = a.norm ? a.norm + bh * a.norm_stride : a.norm;
  h.fresh = a.new_imp ? a.new_imp + bh * a.A : a.new_imp;
  h.path = a.path ? a.path + (long long)b * a.A : a.path;
  h.n = n;
  h.seen = seen;
  return h;
}

// Carries out `count` moves (pair(j): source candidate and target slot) by NT threads: a 16-byte chunk of K or V a thread,
// then eight lanes on each row's numbers (a new row's value norm is a sum over its chunks, in a fixed order).
template <int NT, bool VEC, typename Pair>
__device__ __forceinline__ void ins_move(const InsArgs& a, const InsHead& h, int count, int tid, Pair pair) {
  const int CH = (a.D + 7) / 8, per = 2 * CH;
#pragma unroll 1
  for (int u = tid; u < count * per; u += NT) {
    const int j = u / per, e = u - j * per;
    const bool isv = e >= CH;
    const int ch = 8 * (isv ? e - CH : e);
    int src, dst;
    pair(j, src, dst);
    const bool fresh = src >= h.n;
    const int row = fresh ? (h.path ? h.path[src - h.n] : src - h.n) : src;
    const InsIn from = fresh ? (isv ? h.vn + row * a.vn : h.kn + row * a.kn) : (isv ? (InsIn)h.vc + row * a.vcn : (InsIn)h.kc + row * a.kcn);
    const InsOut to = isv ? h.vc + dst * a.vcn : h.kc + dst * a.kcn;
    if (VEC) {
      *(FE_GLOBAL u32x4*)(to + ch) = *(const FE_GLOBAL u32x4*)(from + ch);
    } else {
      const long long fs = fresh ? (isv ? a.vd : a.kd) : (isv ? a.vcd : a.kcd), ts = isv ? a.vcd : a.kcd;
      for (int d = ch; d < min(ch + 8, a.D); ++d) to[d * ts] = from[d * fs];
    }
  }
#pragma unroll 1
  for (int j = tid >> 3; j < count; j += NT / 8) {
    int src, dst;
    pair(j, src, dst);
    const bool fresh = src >= h.n;
    const int at = src - h.n;
    float s = 0.f;
    if (fresh && h.norm) {
      const InsIn from = h.vn + (long long)(h.path ? h.path[at] : at) * a.vn;
      for (int ch = 8 * (tid & 7); ch < a.D; ch += 64) {
        u16 x[8];
        if (VEC) {
          const u32x4 y = *(const FE_GLOBAL u32x4*)(from + ch);
          __builtin_memcpy(x, &y, 16);
        } else {
          for (int d = 0; d < 8; ++d) x[d] = ch + d < a.D ? from[(ch + d) * a.vd] : (u16)0;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) s += fabsf(a.bf16 ? BF16::to_f32(x[d]) : F16::to_f32(x[d]));
      }
    }
#pragma unroll
    for (int d = 1; d < 8; d *= 2) s += __shfl_xor(s, d);
    if ((tid & 7) == 0) {
      if (h.norm) h.norm[dst] = fresh ? s : h.norm[src];
      h.imp[dst] = fresh ? (h.fresh ? h.fresh[at] : 0.f) : h.imp[src];
      h.pos[dst] = fresh ? h.seen + at : h.pos[src];
    }
  }
}

// Leading nodes of a path that name one of the T tokens, by the whole block. s: one int of LDS.
__device__ __forceinline__ int ins_path_len(const InsArgs& a, const FE_GLOBAL int* path, int* s) {
  if (threadIdx.x == 0) *s = a.A;
  __syncthreads();
  for (int i = threadIdx.x; i < a.A; i += 1024)
    if (path[i] < 0 || path[i] >= a.T) atomicMin(s, i);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*s);
}

// In candidate order, with PER consecutive candidates a thread: hole(i, rank) for each evicted one below F, mover(i, rank)
// for each kept one at or past F, stay(i, rank) for each kept new one below F. Returns the numbers of movers and of
// those that stay. key > thr is kept, and the first `need` of the eq candidates with key == thr.
template <int PER, typename Get, typename Hole, typename Mover, typename Stay>
__device__ __forceinline__ void ins_order(Get get, int n, int M, int F, u32 thr, int need, int eq, int* tmp, Hole hole, Mover mover,
                                          Stay stay, int& moves, int& stays) {
  int eq_before = 0, holes = 0;
  moves = stays = 0;
#pragma unroll 1
  for (int base = 0; base < M; base += 1024 * PER) {
    const int i0 = base + (int)threadIdx.x * PER;
    u32 key[PER];
    int neq = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = i0 + i < M ? get(i0 + i) : 0u;
      neq += i0 + i < M && key[i] == thr ? 1 : 0;
    }
    int rank = 0, total;
    if (need < eq) {
      rank = eq_before + block_exclusive_scan(neq, tmp, total);
      eq_before += total;
    }
    u32 kept = 0;
    int nh = 0, nm = 0, ns = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = i0 + i < M;
      bool k = in && key[i] > thr;
      if (in && key[i] == thr) {
        k = need == eq || rank < need;
        ++rank;
      }
      kept |= k ? 1u << i : 0u;
      nh += in && !k && i0 + i < F ? 1 : 0;
      nm += k && i0 + i >= F ? 1 : 0;
      ns += k && i0 + i >= n && i0 + i < F ? 1 : 0;
    }
    // counts of a round are at most 1024 * PER: 13 bits and more each in two scans
    int at = block_exclusive_scan(nh | (nm << 16), tmp, total);
    int h = holes + (at & 0xffff), m = moves + (at >> 16);
    holes += total & 0xffff;
    moves += total >> 16;
    int s = stays + block_exclusive_scan(ns, tmp, total);
    stays += total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = i0 + i;
      const bool k = (kept >> i) & 1u;
      if (c < M && !k && c < F) hole(c, h++);
      if (k && c >= F) mover(c, m++);
      if (k && c >= n && c < F) stay(c, s++);
    }
  }
}

// Block (KV head, batch row). What bounds it: the trips to memory one after the other (length, keys, rows) and the barrier
// of each drawn victim: one row into 1024 rows of 8 heads 6.4 us, into 8192 rows of 128 heads 7.7, six into 13107 rows of
// 32 heads 12.7; by selection the counts' atomics, 250 into 2000 rows of 16 heads 17.7.
template <bool VEC>
__global__ __launch_bounds__(1024) void insert_few_kernel(const InsArgs args) {
  __shared__ u32 skey[kInsKeys];
  __shared__ int s_src[2 * kInsFew], s_dst[2 * kInsFew];   // moves, then the rows that stay
  __shared__ u32 hist[2 * 2048];
  __shared__ __attribute__((aligned(16))) int tmp[2 * kSelWaves];
  __shared__ SelShared sh;
  __shared__ u32 red_k[2][16];
  __shared__ int red_i[2][16], s_len;
  const InsArgs a = ins_hold(args);
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = (int)blockIdx.x, b = (int)blockIdx.y, bh = b * a.Hkv + hkv;
  const int len = a.length[bh], seen = __builtin_amdgcn_readfirstlane(a.seen[bh]);
  const int n = __builtin_amdgcn_readfirstlane(min(max(len, 0), a.C));
  const InsHead h = ins_head(a, b, hkv, n, seen);
  const int na = h.path ? ins_path_len(a, h.path, &s_len) : a.A;
  const int M = n + na, F = min(M, a.budget), e = M - F;
  const long long held = (long long)seen + na - a.recent;   // first protected position

  int moves = 0, stays = F > n ? F - n : 0;
  if (e > 0) {
    u32 bk = kKeyDrawn;                     // the thread's least key, of equal ones the highest slot
    int bi = -1;
    constexpr int U = 4;
#pragma unroll 1
    for (int base = tid; base < M; base += 1024 * U) {
      float w[U];
      int p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = base + 1024 * u;
        const bool old = i < n;
        const int at = old ? i : 0;
        w[u] = h.imp[at];
        p[u] = h.pos[at];
        if (!old) {
          w[u] = i < M && h.fresh ? h.fresh[i - n] : 0.f;
          p[u] = seen + (i - n);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = base + 1024 * u;
        if (i < M) {
          const u32 key = ins_key(w[u], (i < n ? (long long)p[u] : (long long)seen + (i - n)) >= held);
          skey[i] = key;
          if (key <= bk) bk = key, bi = i;
        }
      }
    }
    if (e <= kInsDraw) {
      int vict = 0x7fffffff;                // lane r: the r-th drawn
#pragma unroll 1
      for (int r = 0; r < e; ++r) {
        const u32 wk = (u32)__builtin_amdgcn_readlane((int)wave_inclusive_min(bk), 63);
        const int wi = __builtin_amdgcn_readlane((int)wave_inclusive_max(bk == wk ? (u32)(bi + 1) : 0u), 63) - 1;
        if (lane == 0) red_k[r & 1][wv] = wk, red_i[r & 1][wv] = wi;
        lds_barrier();
        const u32 k16 = red_k[r & 1][lane & 15];
        const int i16 = red_i[r & 1][lane & 15];
        const u32 K = (u32)__builtin_amdgcn_readlane((int)wave_inclusive_min(k16), 63);
        const int I = __builtin_amdgcn_readlane((int)wave_inclusive_max(k16 == K ? (u32)(i16 + 1) : 0u), 63) - 1;
        if (lane == r) vict = I;
        if (r + 1 < e && ((I & 1023) >> 6) == wv) {
          // the wave finds its thread's next, a key to a lane
          const int i = (I & 1023) + 1024 * lane;
          u32 k = lane < kInsKeys / 1024 && i < M ? skey[i] : kKeyDrawn;
          if (i == I) k = skey[i] = kKeyDrawn;
          const u32 wk2 = (u32)__builtin_amdgcn_readlane((int)wave_inclusive_min(k), 63);
          const int wi2 = __builtin_amdgcn_readlane((int)wave_inclusive_max(k == wk2 && k != kKeyDrawn ? (u32)(i + 1) : 0u), 63) - 1;
          if ((I & 1023) == tid) bk = wk2, bi = wi2;
        }
      }
      // a victim below F leaves a hole, in order; a candidate at or past F that is no victim moves, in order; new rows
      // below F that are no victims stay
      auto drawn = [&](int q) { return __builtin_amdgcn_readlane(vict, q); };
      if (wv == 0) {
        int hole = 0, before = 0, same = 0;
#pragma unroll 1
        for (int q = 0; q < e; ++q) {
          const int x = drawn(q);
          hole += x < vict ? 1 : 0;                       // holes before this one (victims below it are below F)
          before += x >= F && x < F + lane ? 1 : 0;       // victims at or past F before candidate F + lane
          same += x == F + lane ? 1 : 0;
        }
        if (lane < e && vict < F) s_dst[hole] = vict;
        if (lane < e && !same) s_src[lane - before] = F + lane;
      }
      const int past = __popcll(__ballot(vict >= F && vict < M)), fresh = __popcll(__ballot(vict >= n && vict < F));
      moves = e - past;
      for (int i = tid; i < F - n; i += 1024) {
        int before = 0, same = 0;
#pragma unroll 1
        for (int q = 0; q < e; ++q) {
          const int x = drawn(q);
          before += x >= n && x < n + i ? 1 : 0;
          same += x == n + i ? 1 : 0;
        }
        if (!same) s_src[kInsFew + i - before] = s_dst[kInsFew + i - before] = n + i;
      }
      stays -= fresh;
    } else {
      __syncthreads();
      u32 thr;
      int need, eq;
      auto get = [&](int i) -> u32 { return skey[i]; };
      radix_select(get, M, F, 0u, 0xffffffffu, hist, tmp, &sh, thr, need, eq);
      ins_order<4>(get, n, M, F, thr, need, eq, tmp, [&](int i, int r) { s_dst[r] = i; }, [&](int i, int r) { s_src[r] = i; },
                   [&](int i, int r) { s_src[kInsFew + r] = s_dst[kInsFew + r] = i; }, moves, stays);
    }
  } else {
    for (int i = tid; i < stays; i += 1024) s_src[kInsFew + i] = s_dst[kInsFew + i] = n + i;
  }
  __syncthreads();
  ins_move<1024, VEC>(a, h, moves + stays, tid, [&](int j, int& src, int& dst) {
    const int at = j < moves ? j : kInsFew + j - moves;
    src = s_src[at];
    dst = s_dst[at];
  });
  if (tid == 0) {
    a.length[bh] = F;
    a.seen[bh] = seen + na;
  }
}

// Block (KV head, batch row). What bounds it: one CU's reads of the head's keys, once a digit.
__global__ __launch_bounds__(1024) void insert_list_kernel(const InsArgs args) {
  __shared__ u32 hist[2 * 2048];
  __shared__ __attribute__((aligned(16))) int tmp[2 * kSelWaves];
  __shared__ SelShared sh;
  __shared__ int s_len;
  const InsArgs a = ins_hold(args);
  const int hkv = (int)blockIdx.x, b = (int)blockIdx.y, bh = b * a.Hkv + hkv;
  const int n = __builtin_amdgcn_readfirstlane(min(max(a.length[bh], 0), a.C)), seen = __builtin_amdgcn_readfirstlane(a.seen[bh]);
  const InsHead h = ins_head(a, b, hkv, n, seen);
  const int na = h.path ? ins_path_len(a, h.path, &s_len) : a.A;
  const int M = n + na, F = min(M, a.budget);
  const long long held = (long long)seen + na - a.recent;
  FE_GLOBAL int* list = a.lists + (long long)bh * (4 + 2 * (long long)a.P);
  FE_GLOBAL int* dst = list + 4;
  FE_GLOBAL int* src = dst + a.P;
  int moves = 0, stays = F > n ? F - n : 0;
  if (M > F) {
    auto get = [&](int i) -> u32 {
      if (i < n) return ins_key(h.imp[i], h.pos[i] >= held);
      return ins_key(h.fresh ? h.fresh[i - n] : 0.f, (long long)seen + (i - n) >= held);
    };
    u32 thr;
    int need, eq;
    radix_select(get, M, F, 0u, 0xffffffffu, hist, tmp, &sh, thr, need, eq);
    ins_order<8>(get, n, M, F, thr, need, eq, tmp, [&](int i, int r) { dst[r] = i; }, [&](int i, int r) { src[r] = i; },
                 [&](int i, int r) { src[a.P - 1 - r] = dst[a.P - 1 - r] = i; }, moves, stays);
  } else {
    for (int i = threadIdx.x; i < stays; i += 1024) src[a.P - 1 - i] = dst[a.P - 1 - i] = n + i;
  }
  __syncthreads();                          // every wave has read the length
  if (threadIdx.x == 0) {
    list[0] = moves;
    list[1] = stays;
    list[2] = n;
    list[3] = seen;
    a.length[bh] = F;
    a.seen[bh] = seen + na;
  }
}

// What bounds it: HBM, with rows in no order.
template <bool VEC>
__global__ __launch_bounds__(256) void insert_move_kernel(const InsArgs args) {
  const InsArgs a = ins_hold(args);
  const int hkv = (int)blockIdx.y, b = (int)blockIdx.z, bh = b * a.Hkv + hkv;
  const FE_GLOBAL int* list = a.lists + (long long)bh * (4 + 2 * (long long)a.P);
  const int moves = list[0], all = moves + list[1];
  const InsHead h = ins_head(a, b, hkv, list[2], list[3]);
  const FE_GLOBAL int* dsts = list + 4;
  const FE_GLOBAL int* srcs = dsts + a.P;
  // 32 rows a block at a time
#pragma unroll 1
  for (int r0 = 32 * (int)blockIdx.x; r0 < all; r0 += 32 * (int)gridDim.x)
    ins_move<256, VEC>(a, h, min(32, all - r0), threadIdx.x, [&](int j, int& src, int& dst) {
      const int at = r0 + j < moves ? r0 + j : a.P - 1 - (r0 + j - moves);
      src = srcs[at];
      dst = dsts[at];
    });
}

struct InsKernel {
  const void* fn;
  const char* name;
};
const InsKernel kInsKernels[] = {{(const void*)insert_few_kernel<false>, "insert_few_elements"}, {(const void*)insert_few_kernel<true>, "insert_few"},
                                 {(const void*)insert_move_kernel<false>, "insert_move_elements"}, {(const void*)insert_move_kernel<true>, "insert_move"},
                                 {(const void*)insert_list_kernel, "insert_list"}};

void append_insert_resources(std::string& out) {
  for (const auto& e : kInsKernels) {
    hipFuncAttributes attr;
    if (hipFuncGetAttributes(&attr, e.fn) != hipSuccess) continue;
    char buf[512];
    snprintf(buf, sizeof(buf),
             "{\"kernel\":\"%s\",\"registers_per_thread\":%d,\"lds_static_bytes\":%zu,"
             "\"lds_dynamic_bytes\":0,\"scratch_bytes_per_thread\":%zu,\"max_threads_per_block\":%d},",
             e.name, attr.numRegs, (size_t)attr.sharedSizeBytes, (size_t)attr.localSizeBytes, attr.maxThreadsPerBlock);
    out += buf;
  }
}

namespace {
// Whether the few-rows kernel holds all that any lengths can ask for.
bool ins_few(int64_t C, int64_t A, int64_t budget) { return A <= kInsFew && C + A - budget <= kInsFew && C + A <= kInsKeys; }
// Rows that an insertion can write: new ones, and those from past the budget; all below it.
int64_t ins_list(int64_t C, int64_t A, int64_t budget) { return std::min(A + C - budget, budget); }
}  // namespace
}  // namespace fe

using namespace fe;

extern "C" size_t fe_insert_workspace_bytes(int64_t B, int64_t Hkv, int64_t A, int64_t C, int64_t budget) {
  if (B < 1 || Hkv < 1 || A < 0 || C < 1 || budget < 1 || budget > C || B > 65535 || Hkv > 65535 || A > (1LL << 29) ||
      C > (1LL << 30) || B * Hkv > (1LL << 24))
    return 0;
  if (ins_few(C, A, budget)) return 0;
  return (size_t)(B * Hkv) * (size_t)(4 + 2 * ins_list(C, A, budget)) * sizeof(int);
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
  if (C > (1LL << 30) || T > (1LL << 29) || B > 65535 || Hkv > 65535 || B * Hkv > (1LL << 24)) {
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
  const int64_t* st[4] = {k_strides, v_strides, k_cache_strides, v_cache_strides};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (!st[i] || st[i][j] < 0) {
        set_error(std::string(who) + ": null or negative strides");
        return FE_ERR_INVALID;
      }
  const size_t need = fe_insert_workspace_bytes(B, Hkv, A, C, budget);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error(std::string(who) + ": workspace too small; need " + std::to_string(need) + " bytes");
    return FE_ERR_WORKSPACE;
  }
  auto vec = [&](const void* p, const int64_t* s, int64_t N) {
    return D % 8 == 0 && s[3] == 1 && (uintptr_t)p % 16 == 0 && (B <= 1 || s[0] % 8 == 0) && (Hkv <= 1 || s[1] % 8 == 0) &&
           (N <= 1 || s[2] % 8 == 0);
  };
  const bool v16 = vec(k, st[0], T) && vec(v, st[1], T) && vec(k_cache, st[2], C) && vec(v_cache, st[3], C);
  InsArgs a = {};
  auto set = [](auto& to, auto* from) { to = (std::remove_reference_t<decltype(to)>)(uintptr_t)from; };
  set(a.k, k);
  set(a.v, v);
  set(a.kc, k_cache);
  set(a.vc, v_cache);
  set(a.imp, importance);
  set(a.pos, position);
  set(a.norm, value_norm);
  set(a.length, length);
  set(a.seen, seen);
  set(a.new_imp, new_importance);
  set(a.path, path);
  set(a.lists, workspace);
  a.kb = st[0][0], a.kh = st[0][1], a.kn = st[0][2], a.kd = st[0][3];
  a.vb = st[1][0], a.vh = st[1][1], a.vn = st[1][2], a.vd = st[1][3];
  a.kcb = st[2][0], a.kch = st[2][1], a.kcn = st[2][2], a.kcd = st[2][3];
  a.vcb = st[3][0], a.vch = st[3][1], a.vcn = st[3][2], a.vcd = st[3][3];
  a.imp_stride = importance_stride;
  a.pos_stride = position_stride;
  a.norm_stride = value_norm_stride;
  a.T = (int)T;
  a.A = (int)A;
  a.C = (int)C;
  a.D = (int)D;
  a.Hkv = (int)Hkv;
  a.budget = (int)budget;
  a.recent = (int)recent;
  a.P = (int)ins_list(C, A, budget);
  a.bf16 = dtype == FE_DTYPE_BF16;
  hipStream_t stream = (hipStream_t)hip_stream;
  auto launch = [&](const void* fn, dim3 grid, dim3 block) {
    void* args[] = {&a};
    const hipError_t err = hipLaunchKernel(fn, grid, block, args, 0, stream);
    if (err != hipSuccess) set_error(std::string(who) + ": launch: " + hipGetErrorString(err));
    return err == hipSuccess ? FE_OK : FE_ERR_HIP;
  };
  const dim3 heads((unsigned)Hkv, (unsigned)B);
  if (ins_few(C, A, budget)) return launch(kInsKernels[v16].fn, heads, dim3(1024));
  if (int rc = launch(kInsKernels[4].fn, heads, dim3(1024))) return rc;
  if (!a.P) return FE_OK;
  // 32 rows a block, up to some 4096 blocks
  const int64_t blocks = std::min<int64_t>((a.P + 31) / 32, std::max<int64_t>(1, 4096 / (B * Hkv)));
  return launch(kInsKernels[2 + v16].fn, dim3((unsigned)blocks, (unsigned)Hkv, (unsigned)B), dim3(256));
}
