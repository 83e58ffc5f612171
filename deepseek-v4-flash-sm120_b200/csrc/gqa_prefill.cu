// Attention over whole prompts of packed sequences, grouped heads
// (include/dsv4b.h, dsv4b_gqa_prefill), on the tcgen05 tensor cores.
//
//   S = q k^T, P = exp(sm_scale S - m), O = P v, out = O / sum(P)
// with the running maximum m and sum of an online softmax over tiles of 128
// keys.  2 (d_qk + d_v) operations per (query, key) against a few bytes per
// token: bound by the tensor cores, with the exponentials next (a 128 x 128
// tile is 2 * 128^2 (d_qk + d_v) operations, about 1,000 cycles of the tensor
// core at d = 128, and 128^2 exponentials, 1,024 cycles of an SM's 16 a
// cycle).
//
// An item is 256 queries of one head, as two tiles of 128, and the keys they
// see.  While the tensor core multiplies for one tile, four warps do the
// softmax of the other:
//   warps 0-3, 4-7  softmax of tile 0 / 1, a thread per row: S comes from
//                   TMEM, P goes back there over S (16 bits, the A operand
//                   of O += P v).  O is rescaled only when a row's maximum
//                   grew by more than 2^8 (the exact maximum is not needed:
//                   any reference within fp32's reach gives the same
//                   quotient), which after the first tiles is rare;
//   warp 8          issues the MMAs: S_0 S_1, then per key tile O_0 S_0' O_1
//                   S_1', so that each softmax has the other tile's MMAs to
//                   hide behind (starting O when half of P is there was
//                   slower: the warp waits for the other half meanwhile);
//   warp 9          finds the items and loads Q and the K and V rings by TMA
//                   (SWIZZLE_128B), up to an item ahead of the rest;
//   warps 10, 11    V's guards, below.
// TMEM: S_0 [0, 128), S_1 [128, 256), O_0 and O_1 from 256 on.
//
// A CTA stays on its SM and takes its next item from the CTAs that have not
// started yet (cluster launch control), so that the next item's loads and
// first S run under this one's last softmax and output.  A CTA for each item
// spent 6 us of it on its start and end.
//
// Masked keys have P = 0, but 0 * NaN is NaN: a row of V behind the
// sequence's end belongs to another sequence or to nobody, and one behind a
// query's position may hold anything.  Only the last key tiles of a CTA hold
// such rows; there the guard zeroes the rows behind the end and any value
// that is not finite, before the MMA reads them, and notes the rows of the
// latter: a query that does see one has the value added at the end.
//
// Measured (bf16 GEMM of a library on this GPU: 1,663 TFLOP/s in a burst,
// 1,404 for seconds), in a burst at 1,965 MHz and for seconds at the power
// limit's 1,665 to 1,750: one prompt of 16,384, 32 heads over 8, d = 128, 1.82
// ms, 1,210 TFLOP/s, and 2.10; 24 prompts of up to 4,099, 64 heads, 0.75 and
// 0.84; two of up to 2,600, 128 heads of 192 / 128, 0.60 and 0.69.  A pair of
// tiles takes 4,000 cycles: its MMAs need 2,048 of the tensor core (2,330 as
// they are issued), its exponentials 2,048 of their unit.  Both are busy for 48
// % of the time (4,096 tokens), the issue slots for 30: no unit is full, the
// chain from S over P to O of the two tiles is what takes the time.  The
// shorter prompts also lose their edge tiles' masked halves and the items'
// starts and ends.
//
// The list of items needs no lengths on the host: sequence i has the tiles
// from cu_i / 256 + i on, at least as many as it can fill.  The last tiles
// of a sequence, which see most keys, come first.  Heads are taken in groups
// whose K and V stay in L2 (kGroupBytes): 128 heads of 5,000 keys at once
// read theirs from HBM for every tile.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>
#include <type_traits>

#include "dsv4b.h"
#include "dsv4b_kernels.h"
#include "dsv4b_ptx.cuh"
#include "gqa_tc.cuh"

namespace dsv4b {

__device__ int g_gqa_prefill_status;          // kErr* bits on this device
__device__ int g_gqa_prefill_test_stall = 0;  // test hook: Q's first load is withheld

namespace {

constexpr int kM = 128;              // queries of a tile, keys of a tile
constexpr int kQueries = 2 * kM;     // queries of a CTA
constexpr int kThreads = 12 * 32;
constexpr int kSoftmaxRegs = 216, kOtherRegs = 64;  // of 168 at launch: 2 * 216 + 64 <= 3 * 168
constexpr int kMmaWarp = 8, kLoadWarp = 9, kGuardWarp = 10, kGuardWarps = 2;
constexpr int kChunk = kM * 128;     // 128 rows x 64 16-bit columns, swizzled
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxEdge = 4;          // key tiles that some row of an item does not see whole
constexpr int kEdgeRing = 2 * kMaxEdge;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;      // log2 of how far a maximum may be outgrown
// P is 2^kBelow at the maximum, 2^15 at most: in fp16, where the small P of a
// long prompt would else lose digits from 2^-14 and vanish from 2^-25 on, this
// uses its range up to the end (to bf16 it is all the same).
constexpr float kBelow = 7.f;  // and 0x1p-7f at the end
constexpr int64_t kGroupBytes = 40 << 20;  // K and V of the heads that run at a time: a third of L2

struct PrefillArgs {
  int b, h_q, g, causal, total_q, total_k, tiles, group_heads;
  float scale_log2;
  const void* v;
  int64_t stride_v_t, stride_v_h;
  const int32_t* cu_q;
  const int32_t* cu_k;
  void* out;
  int64_t stride_o_t, stride_o_h;
  float* lse;
};

// Ring depths that fit 227 KB beside Q: V in whole tiles (its chunks stay
// side by side), K too, but where only one and a third of its tiles fit (192
// columns): in chunks of 64 columns, each released by itself.
template <int DQK, int DV>
struct Cfg {
  static constexpr int kChunksQ = DQK / 64;
  static constexpr int kQ = 2 * kChunksQ * kChunk;
  static constexpr int kV = (DV / 64) * kChunk;
  static constexpr int kPartsK = DQK == 192 ? 3 : 1;           // of a K tile
  static constexpr int kChunksK = kChunksQ / kPartsK;          // chunks of a part
  static constexpr int kSlotsK = DQK == 192 ? 4 : 6 / kChunksQ;  // parts in the ring
  static constexpr int kStagesV = DQK == 64 ? 6 : 2;
};

// What a CTA works on.
struct Item {
  int q0, rows;       // first query (row of q) and how many, 1 .. 256; 0: no more items
  int k0, n_k;        // the sequence's keys
  int see;            // keys that the first query sees if causal (may be < 0)
  int head;
  __device__ __forceinline__ int limit(int r, int causal) const { return causal ? min(n_k, see + r) : n_k; }
  // key tiles of query tile i
  __device__ __forceinline__ int tiles(int i, int causal) const {
    const int last = min(rows, (i + 1) * kM) - 1;
    return last >= i * kM ? (max(0, limit(last, causal)) + kM - 1) / kM : 0;
  }
  // the first key tile that some row does not see whole
  __device__ __forceinline__ int edge(int causal) const { return max(0, limit(0, causal)) / kM; }
};

struct Shared {
  uint64_t q_full[2], q_empty[2], k_full[6], k_empty[6], v_full[6], v_empty[6], go[kEdgeRing], guard[kEdgeRing];
  uint64_t s_full[2], p_full[2], o_full[2], done;
  uint64_t item_full[2], item_empty[2], next_full;
  alignas(16) uint32_t next[4];  // cluster launch control's answer
  Item item[2];
  uint32_t bad[2][kMaxEdge][4];  // of an item: rows of V with a value that is not finite
  uint32_t tmem;
  int abort;
};
constexpr int kItemReaders = 8 + 1 + 2;  // softmax, MMA and guard warps

template <int DQK, int DV>
constexpr int smem_bytes() {
  using C = Cfg<DQK, DV>;
  return 1024 + C::kQ + C::kSlotsK * C::kChunksK * kChunk + C::kStagesV * C::kV + (int)sizeof(Shared);
}

// Cluster launch control: asks for a CTA of this grid that has not started
// (16 bytes of answer, counted on `bar`), and reads the answer: the CTA's
// number, or -1 when there are none left (then it must not be asked again).
__device__ __forceinline__ void ask_next(uint32_t answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   answer),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int read_next(uint32_t answer) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\tld.shared.b128 a, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tmov.s32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}"
      : "=r"(r)
      : "r"(answer)
      : "memory");
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 bytes to a 32-byte aligned address.
__device__ __forceinline__ void store_32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Bit 15 of a half is set if it is infinite or NaN (its exponent is all ones).
template <typename T>
__device__ __forceinline__ uint32_t maybe_not_finite(uint32_t w) {
  return std::is_same_v<T, __half> ? (w & 0x7C007C00u) + 0x04000400u : (w & 0x7F807F80u) + 0x00800080u;
}
// 0xFFFF in the halves of a word that are infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same_v<T, __half> ? 0x7C007C00u : 0x7F807F80u;
  return __vcmpeq2(w & e, e);
}

template <typename T, int DQK, int DV>
__global__ void __launch_bounds__(kThreads, 1)
gqa_prefill_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, const PrefillArgs a) {
  using C = Cfg<DQK, DV>;
  constexpr int kSlotsK = C::kSlotsK, kStagesV = C::kStagesV, kChunksQ = C::kChunksQ;
  constexpr int kPartsK = C::kPartsK, kPart = C::kChunksK * kChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_s = smem_u32(smem), k_s = q_s + C::kQ, v_s = k_s + kSlotsK * kPart;
  Shared& sh = *reinterpret_cast<Shared*>(smem + C::kQ + kSlotsK * kPart + kStagesV * C::kV);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int causal = a.causal;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], kM);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], kItemReaders);
    }
    for (int i = 0; i < 6; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < kEdgeRing; ++i) {
      mbar_init(&sh.go[i], 1);
      mbar_init(&sh.guard[i], kGuardWarps);
    }
    mbar_init(&sh.done, 1);
    mbar_init(&sh.next_full, 1);
    sh.abort = 0;
    fence_mbarrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* abort = &sh.abort;
  int* status = &g_gqa_prefill_status;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_warp(bar, parity, abort, status); };
  // The w-th item, in every role but the load warp's: rows == 0 at the end
  // (or when a wait gave up).  Released when nothing of it is needed any more.
  auto take = [&](int w) {
    Item it = {};
    if (wait(&sh.item_full[w & 1], (w >> 1) & 1)) it = sh.item[w & 1];
    return it;
  };
  auto release = [&](int w) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_empty[w & 1]);
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      // -------------------------------------------------------------- loads
      const bool withhold = g_gqa_prefill_test_stall != 0;
      int nk = 0, nv = 0, nq[2] = {0, 0}, ge = 0, asks = 0;  // parts of K, tiles of V, Q tiles, edge tiles, asks so far
      bool ok = true;
      auto load_k = [&](const Item& it, int kvh, int j) {
        for (int x = 0; x < kPartsK && ok; ++x, ++nk) {
          const int st = nk % kSlotsK;
          if (nk >= kSlotsK && !(ok = wait(&sh.k_empty[st], (nk / kSlotsK - 1) & 1))) return;
          if (lane == 0) {
            mbar_arrive_expect_tx(&sh.k_full[st], kPart);
            for (int c = 0; c < C::kChunksK; ++c)
              tma_load_3d(k_s + st * kPart + c * kChunk, &tk, (x * C::kChunksK + c) * 64, kvh, it.k0 + j * kM, &sh.k_full[st]);
          }
        }
      };
      int id = blockIdx.x;
      for (int w = 0; ok; ) {
        // the item's sequence: the last i with cu_i / 256 + i <= tile, 32 at a time
        Item it = {};
        if (id >= 0) {
          const int group = id / (a.tiles * a.group_heads), in_group = id - group * (a.tiles * a.group_heads);
          const int heads = min(a.group_heads, a.h_q - group * a.group_heads);
          const int tile = a.tiles - 1 - in_group / heads;
          auto cq = [&](int i) { return min(max(__ldg(a.cu_q + i), 0), a.total_q); };
          int lo = 0, n = a.b;  // it is one of lo .. lo + n - 1
          while (n > 1) {
            const int step = (n + 31) / 32;
            const int i = lo + lane * step;
            const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && (lane == 0 || cq(i) / kQueries + i <= tile));
            const int k = __popc(below) - 1;
            lo += k * step;
            n = min(step, n - k * step);
          }
          const int q_lo = cq(lo), n_q = max(0, cq(lo + 1) - q_lo);
          const int t0 = (tile - (q_lo / kQueries + lo)) * kQueries;
          if (t0 >= 0 && t0 < n_q) {  // (t0 < 0: offsets that do not ascend)
            it.head = group * a.group_heads + in_group % heads;
            it.q0 = q_lo + t0;
            it.rows = min(kQueries, n_q - t0);
            it.k0 = min(max(__ldg(a.cu_k + lo), 0), a.total_k);
            it.n_k = max(0, min(__ldg(a.cu_k + lo + 1), a.total_k) - it.k0);
            it.see = t0 + it.n_k - n_q + 1;
          }
        }
        if (id >= 0 && lane == 0) {  // the next one's number, while this one is loaded
          fence_proxy_async_smem();  // the last answer is read
          mbar_arrive_expect_tx(&sh.next_full, 16);
          ask_next(smem_u32(sh.next), &sh.next_full);
        }
        const bool asked = id >= 0;
        if (it.rows > 0 || !asked) {  // an item, or the end
          if (w >= 2 && !(ok = wait(&sh.item_empty[w & 1], ((w >> 1) - 1) & 1))) break;
          if (lane < 16) (&sh.bad[w & 1][0][0])[lane] = 0;
          __syncwarp();
          if (lane == 0) {
            sh.item[w & 1] = it;
            mbar_arrive(&sh.item_full[w & 1]);
          }
          __syncwarp();
          ++w;
          if (!asked) break;
          const int n0 = it.tiles(0, causal), n1 = it.tiles(1, causal), nt = max(n0, n1), edge = it.edge(causal);
          const int kvh = it.head / a.g;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if ((i ? n1 : n0) == 0) continue;
            if (nq[i] > 0 && !(ok = wait(&sh.q_empty[i], (nq[i] - 1) & 1))) break;
            if (lane == 0 && !(withhold && i == 0)) {
              mbar_arrive_expect_tx(&sh.q_full[i], C::kQ / 2);
              for (int c = 0; c < kChunksQ; ++c)
                tma_load_3d(q_s + i * (C::kQ / 2) + c * kChunk, &tq, c * 64, it.head, it.q0 + i * kM, &sh.q_full[i]);
            }
            ++nq[i];
          }
          if (nt > 0 && ok) load_k(it, kvh, 0);
          for (int j = 0; j < nt && ok; ++j) {  // in the order of use: K_0 V_0 K_1 V_1 ...
            const int st = nv % kStagesV;
            if (nv >= kStagesV && !(ok = wait(&sh.v_empty[st], (nv / kStagesV - 1) & 1))) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&sh.v_full[st], C::kV);
              for (int c = 0; c < DV / 64; ++c)
                tma_load_3d(v_s + st * C::kV + c * kChunk, &tv, c * 64, kvh, it.k0 + j * kM, &sh.v_full[st]);
              if (j >= edge) mbar_arrive(&sh.go[ge % kEdgeRing]);
            }
            if (j >= edge) ++ge;
            ++nv;
            if (j + 1 < nt) load_k(it, kvh, j + 1);
          }
          if (!ok) break;
        }
        if (!(ok = wait(&sh.next_full, asks & 1))) break;
        ++asks;
        id = read_next(smem_u32(sh.next));
        __syncwarp();
      }
      if (*abort) {  // what is in flight lands (or its wait runs out) before the CTA's shared memory goes
        auto land = [&](uint64_t* bar, uint32_t parity) {
          const long long t = clock64();
          while (!mbar_try_wait(smem_u32(bar), parity, 1000u) && clock64() - t < kWaitLimitCycles) {
          }
        };
        for (int x = max(0, nk - kSlotsK); x < nk; ++x) land(&sh.k_full[x % kSlotsK], (x / kSlotsK) & 1);
        for (int x = max(0, nv - kStagesV); x < nv; ++x) land(&sh.v_full[x % kStagesV], (x / kStagesV) & 1);
        for (int i = 0; i < 2; ++i)
          if (nq[i] && !(withhold && i == 0)) land(&sh.q_full[i], (nq[i] - 1) & 1);
        land(&sh.next_full, asks & 1);
      }
    } else if (warp >= kGuardWarp) {
      // -------------------------------------------------------------- guards
      int nv = 0, ge = 0;
      bool ok = true;
      for (int w = 0; ok; ++w) {
        const Item it = take(w);
        if (it.rows == 0) break;
        const int nt = max(it.tiles(0, causal), it.tiles(1, causal)), edge = it.edge(causal);
        for (int j = edge; j < nt; ++j, ++ge) {
          const int x = nv + j, sv = x % kStagesV;
          // `go`: the tile's load is on its way, so its stage's phase is this one
          // (a parity alone does not tell it from the one before the last)
          if (!(ok = wait(&sh.go[ge % kEdgeRing], (ge / kEdgeRing) & 1))) break;
          if (!(ok = wait(&sh.v_full[sv], (x / kStagesV) & 1))) break;
          const int end = it.n_k - j * kM;                           // rows from here on are no keys of ours
          const int from = max(0, it.limit(0, causal) - j * kM);     // rows before it are seen by all
          // A guard takes every second four rows; four loads at once (one by
          // one this took 3 us of every edge tile).
          uint8_t* tile = smem + C::kQ + kSlotsK * kPart + sv * C::kV + (lane & 7) * 16;
          constexpr int kDeep = 4;
          for (int c = 0; c < DV / 64; ++c) {
            for (int r0 = (from & ~7) + (warp - kGuardWarp) * 4 + (lane >> 3); r0 < kM; r0 += kDeep * 8) {
              uint4 v[kDeep];
              uint32_t any = 0;
#pragma unroll
              for (int i = 0; i < kDeep; ++i) {
                const int r = r0 + i * 8;
                v[i] = r < end && r < kM ? *reinterpret_cast<const uint4*>(tile + c * kChunk + r * 128) : make_uint4(0, 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < kDeep; ++i)
                any |= maybe_not_finite<T>(v[i].x) | maybe_not_finite<T>(v[i].y) | maybe_not_finite<T>(v[i].z) |
                       maybe_not_finite<T>(v[i].w);
              if (any & 0x80008000u) {
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                  const int r = r0 + i * 8;
                  const uint4 m = make_uint4(not_finite<T>(v[i].x), not_finite<T>(v[i].y), not_finite<T>(v[i].z),
                                             not_finite<T>(v[i].w));
                  if (r >= from && (m.x | m.y | m.z | m.w)) {
                    *reinterpret_cast<uint4*>(tile + c * kChunk + r * 128) =
                        make_uint4(v[i].x & ~m.x, v[i].y & ~m.y, v[i].z & ~m.z, v[i].w & ~m.w);
                    atomicOr(&sh.bad[w & 1][j - edge][r >> 5], 1u << (r & 31));
                  }
                }
              }
#pragma unroll
              for (int i = 0; i < kDeep; ++i) {
                const int r = r0 + i * 8;
                if (r >= end && r < kM) *reinterpret_cast<uint4*>(tile + c * kChunk + r * 128) = make_uint4(0, 0, 0, 0);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.guard[ge % kEdgeRing]);
        }
        nv += nt;
        release(w);
      }
    } else {
      // -------------------------------------------------------------- MMAs
      constexpr uint32_t idesc_s = idesc_of<T>(kM, false), idesc_o = idesc_of<T>(DV, true);
      int nk = 0, nv = 0, nq[2] = {0, 0}, np[2] = {0, 0}, ge = 0;
      bool ok = true;
      // The tensor core holds few MMAs in advance, so what this warp executes
      // between them is tensor time (8 cycles an MMA of 64 for the commits and
      // branches alone): a descriptor is a low word, made once for a run of
      // MMAs and stepped, and one high word for all; one elected region holds
      // a tile's O and next S.  (`at`: not hoisted out of the loops, where the
      // descriptors would fill the registers many times over.)
      auto at = [](uint32_t saddr, uint32_t lbo) {
        uint32_t lo = desc_low(saddr, lbo);
        asm volatile("" : "+r"(lo));
        return lo;
      };
      // the K parts from nk on have landed
      auto keys = [&]() {
#pragma unroll
        for (int x = 0; x < kPartsK && ok; ++x) ok = wait(&sh.k_full[(nk + x) % kSlotsK], ((nk + x) / kSlotsK) & 1);
      };
      // S_i = Q_i K^T from them, by the elected thread; `last`: they are released
      auto scores = [&](int i, bool last) {
#pragma unroll
        for (int x = 0; x < kPartsK; ++x) {
          const int st = (nk + x) % kSlotsK;
#pragma unroll
          for (int c = 0; c < C::kChunksK; ++c) {
            const int chunk = x * C::kChunksK + c;
            const uint32_t q_at = at(q_s + i * (C::kQ / 2) + chunk * kChunk, 16), k_at = at(k_s + st * kPart + c * kChunk, 16);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ss(tmem + i * kM, q_at + kk * 2, k_at + kk * 2, kSw128High, idesc_s, (chunk | kk) != 0);
          }
          if (last) umma_commit(&sh.k_empty[st]);
        }
        umma_commit(&sh.s_full[i]);
      };
      for (int w = 0; ok; ++w) {
        const Item it = take(w);
        if (it.rows == 0) break;
        const int n[2] = {it.tiles(0, causal), it.tiles(1, causal)}, nt = max(n[0], n[1]), edge = it.edge(causal);
        release(w);
        if (nt == 0) continue;
        keys();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!ok || n[i] == 0) continue;
          if (!(ok = wait(&sh.q_full[i], nq[i] & 1))) continue;
          ++nq[i];
          if (elect_one()) {
            scores(i, i == 1 || n[1] == 0);
            if (n[i] == 1) umma_commit(&sh.q_empty[i]);
          }
          __syncwarp();
        }
        nk += kPartsK;
        for (int j = 0; j < nt && ok; ++j) {
          // all that this tile's MMAs need beside P, before P's waits
          const int sv = nv % kStagesV;
          ok = wait(&sh.v_full[sv], (nv / kStagesV) & 1);
          if (ok && j >= edge) {
            ok = wait(&sh.guard[ge % kEdgeRing], (ge / kEdgeRing) & 1);
            ++ge;
          }
          if (ok && j + 1 < nt) keys();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!ok || j >= n[i]) continue;
            if (!(ok = wait(&sh.p_full[i], np[i] & 1))) continue;
            ++np[i];
            tc_fence_after();
            if (elect_one()) {
              const uint32_t v_at = at(v_s + sv * C::kV, kChunk);
#pragma unroll
              for (int kk = 0; kk < kM / 16; ++kk)  // O_i += P_i V
                umma_ts(tmem + 256 + i * DV, tmem + i * kM + kk * 8, v_at + kk * 128, kSw128High, idesc_o, (j | kk) != 0);
              if (i == 1 || j >= n[1]) umma_commit(&sh.v_empty[sv]);
              if (j + 1 < n[i]) {
                scores(i, i == 1 || j + 1 >= n[1]);
                if (j + 2 == n[i]) umma_commit(&sh.q_empty[i]);
              } else {
                umma_commit(&sh.o_full[i]);
              }
            }
            __syncwarp();
          }
          ++nv;
          if (j + 1 < nt) nk += kPartsK;
        }
      }
      // every MMA has completed before TMEM is freed
      if (elect_one()) umma_commit(&sh.done);
      __syncwarp();
      const long long t = clock64();
      while (!mbar_try_wait(smem_u32(&sh.done), 0, 1000u) && clock64() - t < kWaitLimitCycles) {
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------------------------------------------------------- softmax
    const int i = warp >> 2;  // query tile
    const int r = i * kM + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + lanes + i * kM, o_t = tmem + lanes + 256 + i * DV;
    const float c = a.scale_log2;
    int ns = 0, no = 0, ge = 0;  // S tiles, items with any, edge tiles so far
    bool ok = true;
    for (int w = 0; ok; ++w) {
      const Item it = take(w);
      if (it.rows == 0) break;
      const int mine = it.tiles(i, causal), nt = max(it.tiles(0, causal), it.tiles(1, causal)), edge = it.edge(causal);
      const int lim = it.limit(r, causal), lim0 = it.limit(i * kM, causal);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < mine; ++j, ++ns) {
        if (!(ok = wait(&sh.s_full[i], ns & 1))) break;
        tc_fence_after();
        float s[kM];
#pragma unroll
        for (int x = 0; x < kM; x += 32) tmem_ld32(s_t + x, *reinterpret_cast<float(*)[32]>(&s[x]));
        tc_wait_ld();
        // 32 columns at a time: those that some row of the warp does not see are
        // masked, and from `seen` on no row of it sees any
        int seen = kM;
        if (j * kM + kM > lim0) {
          const int left = lim - j * kM, least = __shfl_sync(0xffffffffu, left, 0);
          seen = __shfl_sync(0xffffffffu, left, 31);
#pragma unroll
          for (int x = 0; x < kM; x += 32) {
            if (x + 32 > least) {
#pragma unroll
              for (int e = 0; e < 32; ++e) s[x + e] = x + e < left ? s[x + e] : -INFINITY;
            }
          }
        }
        float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int x = 4; x + 8 <= kM; x += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = max3(t[e], s[x + 2 * e], s[x + 2 * e + 1]);
        }
        t[0] = max3(t[0], s[kM - 4], s[kM - 3]);
        t[1] = max3(t[1], s[kM - 2], s[kM - 1]);
        const float top = fmaxf(max3(t[0], t[1], t[2]), t[3]);
        const bool grew = (top - m) * c > kRescale;  // from -inf: always
        if (__any_sync(0xffffffffu, grew)) {
          const float f = grew ? fast_exp2((m - top) * c) : 1.f;
          if (grew) m = top;
          l *= f;
          if (j > 0) {  // the MMAs of the tile before are complete: this tile's S came after them
#pragma unroll
            for (int x = 0; x < DV; x += 16) {  // (beside S's 128 registers)
              float o[16];
              tmem_ld16(o_t + x, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st16(o_t + x, o);
            }
          }
        }
        const float mc = kBelow - (m == -INFINITY ? 0.f : m * c);
        const uint64_t cc = pair(c, c), mm = pair(mc, mc);
        uint64_t l2[2] = {0, 0};  // two pairs of zeros
#pragma unroll
        for (int x = 0; x < kM; x += 32) {
          float p[16];
          if (x >= seen) {
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = 0.f;
            tmem_st16(s_t + x / 2, p);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 u = unpair(fma2(pair(s[x + 2 * e], s[x + 2 * e + 1]), cc, mm));
            u.x = fast_exp2(u.x);
            u.y = fast_exp2(u.y);
            l2[e & 1] = add2(l2[e & 1], pair(u.x, u.y));
            p[e] = __uint_as_float(pack16<T>(u.x, u.y));
          }
          tmem_st16(s_t + x / 2, p);
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.p_full[i]);
        const float2 sum = unpair(add2(l2[0], l2[1]));
        l += sum.x + sum.y;
      }
      if (!ok) break;
      if (mine > 0) {
        if (!(ok = wait(&sh.o_full[i], no & 1))) break;
        ++no;
      }
      // rows of V that were kept out of the products, for those who see them
      bool bad = false;
      for (int j = edge; j < mine && ok; ++j) {
        const int x = ge + j - edge;
        ok = wait(&sh.guard[x % kEdgeRing], (x / kEdgeRing) & 1);
        const uint32_t* b = sh.bad[w & 1][j - edge];
        bad |= (b[0] | b[1] | b[2] | b[3]) != 0;
      }
      if (!ok) break;
      ge += max(0, nt - edge);
      tc_fence_after();
      const bool live = r < it.rows;
      const bool none = lim <= 0;
      const float inv = 1.f / l;
      // whole 32-byte sectors where every row starts on one
      const bool wide = ((reinterpret_cast<uintptr_t>(a.out) & 31) | ((a.stride_o_t | a.stride_o_h) & 15)) == 0;
      T* out = static_cast<T*>(a.out) + (int64_t)(it.q0 + r) * a.stride_o_t + (int64_t)it.head * a.stride_o_h;
#pragma unroll
      for (int x = 0; x < DV; x += 32) {
        float o[32];
        if (mine > 0) {
          tmem_ld32(o_t + x, o);
          tc_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = none ? 0.f : o[e] * inv;
        if (bad) {
          for (int j = edge; j < mine; ++j)
            for (int k = 0; k < 4; ++k)
              for (uint32_t bits = sh.bad[w & 1][j - edge][k]; bits; bits &= bits - 1) {
                const int t = j * kM + k * 32 + __ffs(bits) - 1;
                if (t >= lim) continue;
                const T* v = static_cast<const T*>(a.v) + (int64_t)(it.k0 + t) * a.stride_v_t +
                             (int64_t)(it.head / a.g) * a.stride_v_h + x;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float f = static_cast<float>(v[e]);
                  if (!(fabsf(f) < INFINITY)) o[e] += f;
                }
              }
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = pack16<T>(o[e + 2 * k], o[e + 2 * k + 1]);
            if (wide) {
              store_32(out + x + e, v);
            } else {
              *reinterpret_cast<uint4*>(out + x + e) = make_uint4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<uint4*>(out + x + e + 8) = make_uint4(v[4], v[5], v[6], v[7]);
            }
          }
        }
      }
      if (live) a.lse[(int64_t)(it.q0 + r) * a.h_q + it.head] = none ? -INFINITY : (m * c + log2f(l * 0x1p-7f)) * kLn2;
      tc_fence_before();  // O is read before the arrival that lets the next item's MMAs write it
      release(w);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// [tokens][heads][d] of 16 bits, boxes of 128 tokens x 64 columns of a head.
bool make_map(CUtensorMap* m, const void* base, int64_t tokens, int heads, int d, int64_t stride_t, int64_t stride_h,
              int dtype) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)stride_h * 2, (cuuint64_t)stride_t * 2};
  const cuuint32_t box[3] = {64, 1, kM};
  const cuuint32_t es[3] = {1, 1, 1};
  return enc(m, dtype == DSV4B_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DQK, int DV>
cudaError_t launch(const dsv4b_gqa_prefill_params& p, cudaStream_t stream, int* bad_arg) {
  CUtensorMap tq, tk, tv;
  // without a single key nothing is loaded: any valid map will do
  const bool keys = p.total_k > 0;
  if (!make_map(&tq, p.q, p.total_q, p.h_q, DQK, p.stride_q_t, p.stride_q_h, p.dtype) ||
      !make_map(&tk, keys ? p.k : p.q, keys ? p.total_k : 1, keys ? p.h_kv : 1, DQK, keys ? p.stride_k_t : DQK,
                keys ? p.stride_k_h : DQK, p.dtype) ||
      !make_map(&tv, keys ? p.v : p.q, keys ? p.total_k : 1, keys ? p.h_kv : 1, DV, keys ? p.stride_v_t : DV,
                keys ? p.stride_v_h : DV, p.dtype)) {
    *bad_arg = 1;
    return cudaErrorInvalidValue;
  }
  PrefillArgs a = {};
  a.b = p.b;
  a.h_q = p.h_q;
  a.g = p.h_q / p.h_kv;
  a.causal = p.causal;
  a.total_q = (int)p.total_q;
  a.total_k = (int)p.total_k;
  a.tiles = (int)p.total_q / kQueries + p.b;
  const int64_t head_bytes = p.total_k * (DQK + DV) * 2;
  const int64_t kv_heads = head_bytes > 0 ? kGroupBytes / head_bytes : p.h_kv;
  a.group_heads = a.g * (int)(kv_heads < 1 ? 1 : kv_heads > p.h_kv ? p.h_kv : kv_heads);
  a.scale_log2 = p.sm_scale * kLog2e;
  a.v = p.v;
  a.stride_v_t = p.stride_v_t;
  a.stride_v_h = p.stride_v_h;
  a.cu_q = p.cu_seqlens_q;
  a.cu_k = p.cu_seqlens_k;
  a.out = p.out;
  a.stride_o_t = p.stride_o_t;
  a.stride_o_h = p.stride_o_h;
  a.lse = p.lse;
  constexpr int smem = smem_bytes<DQK, DV>();
  static_assert(smem <= 227 * 1024, "prefill kernel shared memory");
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !done[dev]) {
    e = cudaFuncSetAttribute(gqa_prefill_kernel<T, DQK, DV>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  gqa_prefill_kernel<T, DQK, DV><<<(unsigned)((int64_t)a.tiles * p.h_q), kThreads, smem, stream>>>(tq, tk, tv, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gqa_prefill(const dsv4b_gqa_prefill_params& p, cudaStream_t stream, int* bad_arg) {
  if (p.dtype == DSV4B_BF16) {
    if (p.d_qk == 64) return launch<__nv_bfloat16, 64, 64>(p, stream, bad_arg);
    if (p.d_qk == 128) return launch<__nv_bfloat16, 128, 128>(p, stream, bad_arg);
    return launch<__nv_bfloat16, 192, 128>(p, stream, bad_arg);
  }
  if (p.d_qk == 64) return launch<__half, 64, 64>(p, stream, bad_arg);
  if (p.d_qk == 128) return launch<__half, 128, 128>(p, stream, bad_arg);
  return launch<__half, 192, 128>(p, stream, bad_arg);
}

cudaError_t read_gqa_prefill_status(int* flags, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(flags, g_gqa_prefill_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return e;
  if ((e = cudaStreamSynchronize(stream)) != cudaSuccess) return e;
  static const int zero = 0;
  return cudaMemcpyToSymbolAsync(g_gqa_prefill_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
}

cudaError_t set_gqa_prefill_test_stall(int stall) {
  return cudaMemcpyToSymbol(g_gqa_prefill_test_stall, &stall, sizeof(stall));
}

}  // namespace dsv4b
