// Attention over the 8-bit grouped-query cache, and the attention weights of
// its positions (include/dsv4b.h, dsv4b_gqa_decode and
// dsv4b_gqa_attention_weights).
//
//   s[r][t] = sm_scale * k_scale * sum_d q[r][d] * k[t][d]
//   out[r]  = sum_t exp(s[r][t] - lse[r]) * v_scale * v[t]
// for the rows r = (query, head) that share a KV head: h_q / h_kv * s_q of
// them, few against the positions.  Every cached byte is used for all rows
// at once and only once, so the kernel is bound by the cache's bytes.
//
// Work.  A unit is 32 positions of one (sequence, KV head, group of 16
// rows).  All units stand in one list, and every warp of the grid (one CTA
// of eight warps per SM) takes an equal, contiguous piece of it, so ragged
// batches balance without a plan made ahead.  A warp runs the softmax of its
// piece by itself: no barrier until its CTA's end, where pieces of one
// (sequence, head, group) are joined; those that reach over CTAs are joined
// by a second kernel.
//
// Loads.  Each warp has its own ring of two stages (32 positions of K and of
// V, 8 KB at d = 128), filled by TMA tiled loads that swizzle the rows and
// counted on an mbarrier: 128 KB are in flight on an SM, without a register
// or an issue slot spent on them.
//
// Products.  mma.sync m16n8k16 with fp16 operands, the 16 rows as M.  The
// operands of tcgen05 would have to stand in shared memory in their final
// type, so e4m3 would be widened into shared memory (twice its bytes written
// and read again) for 16 useful rows of 128; mma.sync takes them from
// registers, where an e4m3 pair becomes an fp16 pair (exactly) in one
// instruction, and its rate is far above what the loads can feed.  The order
// of d in q.k and of the positions in p.v is free, so the fragments are
// built from 16-byte pieces of whole rows:
//   K: thread (j, c) of a quad reads bytes [16c, 16c + 16) (and 64 further)
//      of position perm(j): four k-steps, with q laid out to match;
//   V: it reads 16 bytes of column piece col(j) of the four positions whose
//      p it holds, and interleaves the bytes of two positions.
// perm and col make every such read free of bank conflicts (below).
//
// Numbers.  q is scaled by a power of two per row so that fp16 holds it
// (bf16 has fewer digits; what lies 2^-27 below the row's largest is lost).
// p <= 1 is rounded to fp16 for p.v (2^-11 of each term), sums and the
// softmax's denominator are fp32 of the unrounded p.  The accumulator is
// kept in units of the current block's v_scale and rescaled when that or
// the running maximum changes, so that no scale enters an fp16.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>
#include <type_traits>

#include "dsv4b.h"
#include "dsv4b_kernels.h"
#include "dsv4b_ptx.cuh"

namespace dsv4b {

__device__ int g_gqa_status;  // kErr* bits of the grouped-query kernels on this device
// Test hook (dsv4b_set_test_stall): when set, the first load of every CTA
// is withheld, so that the first wait runs out.
__device__ int g_gqa_test_stall = 0;

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 32;   // positions of a unit
constexpr int kRows = 16;   // rows of a group (M of the MMA)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct GqaArgs {
  const void* q;
  int64_t stride_q_b, stride_q_s, stride_q_h;
  int s_q, h_q, h_kv, g, groups;  // g = h_q / h_kv; groups of 16 rows per KV head
  float scale_log2;               // sm_scale * log2(e)
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int64_t stride_table;
  int table_width, num_blocks, page, page_shift, b;
  const int32_t* ctx;
  // decode
  void* out;
  int64_t stride_o_b, stride_o_s, stride_o_h;
  float* lse;
  float* ws;
  // attention weights
  const float* lse_in;
  float* weights;
  int64_t stride_w_b, stride_w_h;
  int width, accumulate;
};

// Positions of sequence i that the call reads, and its context length.
__device__ __forceinline__ int held_len(const GqaArgs& a, int i) {
  const int64_t room = (int64_t)a.table_width * a.page;
  return (int)min((int64_t)max(__ldg(a.ctx + i), 0), room);
}
__device__ __forceinline__ int units_of(const GqaArgs& a, int i) {
  return max(1, (held_len(a, i) + kUnit - 1) / kUnit);  // an empty sequence has its outputs written too
}

// ------------------------------------------------------------------ layouts
// Rows of d bytes, swizzled by TMA: 16-byte piece p of row r lies at
// p ^ (r & 7) (128-byte rows) or p ^ ((r >> 1) & 3) (64-byte rows).
template <int D>
struct Lay;
template <>
struct Lay<128> {
  static constexpr int kStages = 2;
  // A quarter of a warp's 16-byte reads (8 threads) is j, j + 1 with all c
  // for K, and for V.  Rows that differ in bit 2 swap the halves of the row,
  // so K wants perm(2j), perm(2j + 1) four apart and V wants col(2j),
  // col(2j + 1) four pieces apart.
  static __device__ __forceinline__ int perm(int j) { return (j >> 1) | ((j & 1) << 2); }
  static __device__ __forceinline__ int col(int j) { return ((j >> 1) | ((j & 1) << 2)) * 16; }  // dims [col, col + 16)
  static __device__ __forceinline__ uint32_t piece(int row, int p) { return row * 128 + ((p ^ (row & 7)) << 4); }
};
template <>
struct Lay<64> {
  static constexpr int kStages = 4;
  // Two rows share 128 bytes, the odd one in the upper half: K wants
  // perm(2j), perm(2j + 1) of different parity, V (8-byte reads, 16 threads
  // at once) wants perm(0), perm(2), perm(4), perm(6) of changing parity.
  static __device__ __forceinline__ int perm(int j) { return j ^ ((j >> 1) & 1); }
  static __device__ __forceinline__ int col(int j) { return j * 8; }  // dims [col, col + 8)
  static __device__ __forceinline__ uint32_t piece(int row, int p) { return row * 64 + ((p ^ ((row >> 1) & 3)) << 4); }
};

__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds_v2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Two e4m3 (low byte first) as two fp16, exactly.
__device__ __forceinline__ uint32_t widen(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four consecutive values of a 16-bit row.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
  if constexpr (std::is_same_v<T, __half>) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
  }
}

// A row's address in q (row r of the KV head: query r / g, head r % g).
template <typename T>
__device__ __forceinline__ const T* q_row(const GqaArgs& a, int b, int kvh, int r) {
  return static_cast<const T*>(a.q) + (int64_t)b * a.stride_q_b + (int64_t)(r / a.g) * a.stride_q_s +
         (int64_t)(kvh * a.g + r % a.g) * a.stride_q_h;
}

// The q fragments of 16 rows from row r0 on: thread (j, c) holds rows j and
// j + 8, for k-step 4 h + s the dims 16 (4 h + c) + 4 s + {0, 1, 2, 3}, the
// same that it reads of K.  Rows past `rows` are zero.  factor[i] is what a
// product is multiplied by: the row's power of two and the softmax scale.
template <typename T, int D>
__device__ __forceinline__ void load_q(const GqaArgs& a, int b, int kvh, int r0, int rows, uint32_t (&q)[D / 16][4],
                                       float (&factor)[2]) {
  const int lane = threadIdx.x & 31, j = lane >> 2, c = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + j + 8 * i;
    const bool live = r < rows;
    const T* p = live ? q_row<T>(a, b, kvh, r) : nullptr;
    float4 f[D / 16];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      f[s] = live ? load4(p + (s >> 2) * 64 + c * 16 + (s & 3) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      top = fmaxf(top, fmaxf(fmaxf(fabsf(f[s].x), fabsf(f[s].y)), fmaxf(fabsf(f[s].z), fabsf(f[s].w))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the row's largest value becomes 2^13 .. 2^14 (an infinite one stays so)
    const int e = min(max((int)(__float_as_uint(top) >> 23), 40), 240) - 127 - 13;
    const float up = __uint_as_float((uint32_t)(127 - e) << 23);
    factor[i] = a.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      q[s][i] = pack_half(f[s].x * up, f[s].y * up);
      q[s][2 + i] = pack_half(f[s].z * up, f[s].w * up);
    }
  }
}

// q.k of the 16 rows with the 32 positions of a stage: s[nt][0, 1] row j,
// s[nt][2, 3] row j + 8, positions 8 nt + perm(2 c), 8 nt + perm(2 c + 1).
template <int D>
__device__ __forceinline__ void score_unit(uint32_t k_stage, const uint32_t (&q)[D / 16][4], float (&s)[4][4]) {
  const int lane = threadIdx.x & 31, j = lane >> 2, c = lane & 3;
#pragma unroll
  for (int nt = 0; nt < 4; ++nt) {
    s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 w = lds_v4(k_stage + Lay<D>::piece(nt * 8 + Lay<D>::perm(j), 4 * h + c));
      mma_f16(s[nt], q[4 * h + 0], widen(w.x & 0xFFFFu), widen(w.x >> 16));
      mma_f16(s[nt], q[4 * h + 1], widen(w.y & 0xFFFFu), widen(w.y >> 16));
      mma_f16(s[nt], q[4 * h + 2], widen(w.z & 0xFFFFu), widen(w.z >> 16));
      mma_f16(s[nt], q[4 * h + 3], widen(w.w & 0xFFFFu), widen(w.w >> 16));
    }
  }
}

// ------------------------------------------------------------------ the list
struct Place {
  int b, kvh, grp;  // sequence, KV head, group of rows
  int u, nu;        // unit in it, and how many it has
};

struct ListShared {
  long long sum[kWarps];
  long long total;
  int b[kWarps + 1];
  long long u[kWarps + 1];
};

// Every thread sums a run of sequences, the sums are scanned, and the thread
// whose run holds a wanted position walks to it.  `want(i, total)` is the
// i-th wanted position; one at or past the total is not placed (b = -1).
template <typename Want>
__device__ __forceinline__ void find_places(const GqaArgs& a, int per_seq, int n, ListShared& sh, Want want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (a.b + kThreads - 1) / kThreads;
  const int i0 = min(a.b, tid * run), i1 = min(a.b, i0 + run);
  long long sum = 0;
  for (int i = i0; i < i1; ++i) sum += units_of(a, i);
  sum *= per_seq;
  long long incl = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.sum[warp] = incl;
  if (tid < n) sh.b[tid] = -1;
  __syncthreads();
  long long pre = incl - sum, total = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) pre += sh.sum[i];
    total += sh.sum[i];
  }
  if (tid == 0) sh.total = total;
  for (int k = 0; k < n; ++k) {
    const long long x = want(k, total);
    if (x >= pre && x < pre + sum) {
      long long at = pre;
      for (int i = i0; i < i1; ++i) {
        const long long m = (long long)units_of(a, i) * per_seq;
        if (x < at + m) {
          sh.b[k] = i;
          sh.u[k] = x - at;
          break;
        }
        at += m;
      }
    }
  }
  __syncthreads();
}

// Position x of `parts` equal pieces of a list: where piece i begins, and
// which piece holds x.
__device__ __forceinline__ long long piece_begin(long long total, long long i, long long parts) {
  return total * i / parts;
}
__device__ __forceinline__ int piece_of(long long total, long long x, long long parts) {
  return (int)(((x + 1) * parts - 1) / total);
}

// ------------------------------------------------------------------ loading
// A warp's ring: its own stages, one mbarrier each.  The load cursor runs
// kStages units ahead of the one that computes.
template <int D, bool WITH_V>
struct Ring {
  static constexpr int kStages = WITH_V ? Lay<D>::kStages : 2 * Lay<D>::kStages;
  static constexpr int kTile = kUnit * D;                  // bytes of K (or V) of a unit
  static constexpr int kStage = kTile * (WITH_V ? 2 : 1);
  static constexpr int kBytes = kStages * kStage;
};

// The block ids of 16 units of a sequence, one per 16 positions, in the
// lanes; `base` is the first unit's number (-1: none held).
struct Pages {
  int id, base, b;
};

__device__ __forceinline__ void fetch_pages(const GqaArgs& a, Pages& p, int b, int u, int len) {
  if (p.b == b && p.base >= 0 && u >= p.base && u < p.base + 16) return;
  const int lane = threadIdx.x & 31;
  p.b = b;
  p.base = u & ~15;
  const long long t = ((long long)p.base * 2 + lane) * 16;
  p.id = -1;
  if (t < len) {
    const int id = __ldg(a.table + (int64_t)b * a.stride_table + (int)(t >> a.page_shift));
    if (id >= 0 && id < a.num_blocks) p.id = id;
  }
}

// Issues the loads of unit u into a stage; returns, in every lane, which of
// the unit's two halves of 16 positions are held (bits 0, 1) and, in lanes
// 0-3, the scales of K (half 0, 1) and V (half 0, 1).
template <int D, bool WITH_V>
__device__ __forceinline__ int load_unit(const GqaArgs& a, const CUtensorMap* tk, const CUtensorMap* tv, Pages& pages,
                                         int b, int kvh, int u, int len, uint32_t stage, uint64_t* bar, float& scale,
                                         bool withhold) {
  using R = Ring<D, WITH_V>;
  const int lane = threadIdx.x & 31;
  fetch_pages(a, pages, b, u, len);
  const int i = (u - pages.base) * 2;
  const int id0 = __shfl_sync(0xffffffffu, pages.id, i), id1 = __shfl_sync(0xffffffffu, pages.id, i + 1);
  const int my = lane & 1 ? id1 : id0;
  scale = 1.f;
  if (lane < (WITH_V ? 4 : 2) && my >= 0)
    scale = __ldg((lane < 2 ? a.k_scale : a.v_scale) + (int64_t)my * a.h_kv + kvh);
  const int held = (id0 >= 0 ? 1 : 0) | (id1 >= 0 ? 2 : 0);
  if (lane == 0 && !withhold) {
    const int off = (u * kUnit) & (a.page - 1);
    if (a.page >= kUnit) {  // one block holds the unit (its second half too, read or not)
      mbar_arrive_expect_tx(bar, id0 >= 0 ? R::kStage : 0);
      if (id0 >= 0) {
        tma_load_4d(stage, tk, 0, off, kvh, id0, bar);
        if constexpr (WITH_V) tma_load_4d(stage + R::kTile, tv, 0, off, kvh, id0, bar);
      }
    } else {
      mbar_arrive_expect_tx(bar, __popc(held) * (R::kStage / 2));
      if (id0 >= 0) {
        tma_load_4d(stage, tk, 0, 0, kvh, id0, bar);
        if constexpr (WITH_V) tma_load_4d(stage + R::kTile, tv, 0, 0, kvh, id0, bar);
      }
      if (id1 >= 0) {
        tma_load_4d(stage + R::kTile / 2, tk, 0, 0, kvh, id1, bar);
        if constexpr (WITH_V) tma_load_4d(stage + R::kTile + R::kTile / 2, tv, 0, 0, kvh, id1, bar);
      }
    }
  }
  return held;
}

// ------------------------------------------------------------------ decode
template <int D>
struct DecodeShared {
  uint64_t full[kWarps][Ring<D, true>::kStages];
  ListShared list;
  // Pieces of one (sequence, head, group) that a warp began or ended with:
  // [warp][first or last piece].  The values of a last one lie in the warp's
  // ring, which it no longer needs.
  int id[kWarps][2];        // (b, kvh, grp) as one number, -1: none
  int from[kWarps][2], to[kWarps][2], nu[kWarps][2];
  float m[kWarps][2][kRows], l[kWarps][2][kRows];
  int abort;
};
template <int D>
constexpr int decode_smem() {
  return 1024 + kWarps * Ring<D, true>::kBytes + kWarps * kRows * D * 4 + (int)sizeof(DecodeShared<D>);
}

// Workspace: [CTA][2] records of {id, last CTA, begins here, rows},
// m[16], l[16], o[16][D]; the first is a piece whose beginning lies in an
// earlier CTA, the second one that goes on in the next.
template <int D>
struct Partial {
  int id, last, begins, ends;
  float m[kRows], l[kRows];
  float o[kRows * D];
};

__device__ __forceinline__ void store_row16(__nv_bfloat16* p, const float* v, int n) {
  for (int i = 0; i < n; i += 8) {
    uint4 w;
    uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[i + 2 * k], v[i + 2 * k + 1]);
      x[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p + i) = w;
  }
}
__device__ __forceinline__ void store_row16(__half* p, const float* v, int n) {
  for (int i = 0; i < n; i += 8) {
    uint4 w;
    uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = pack_half(v[i + 2 * k], v[i + 2 * k + 1]);
    *reinterpret_cast<uint4*>(p + i) = w;
  }
}

template <typename T>
__device__ __forceinline__ T* out_row(const GqaArgs& a, int b, int kvh, int r) {
  return static_cast<T*>(a.out) + (int64_t)b * a.stride_o_b + (int64_t)(r / a.g) * a.stride_o_s +
         (int64_t)(kvh * a.g + r % a.g) * a.stride_o_h;
}
__device__ __forceinline__ float* lse_at(const GqaArgs& a, int b, int kvh, int r) {
  return a.lse + ((int64_t)b * a.h_q + kvh * a.g + r % a.g) * a.s_q + r / a.g;
}

// Joins n pieces of one (sequence, head, group), in order, by all threads:
// piece i has maxima and sums ml(i) (m[16] then l[16]) and values o(i)
// [16][D].  Writes the result, or the joined piece to `part`.
template <typename T, int D, typename ML, typename O>
__device__ __forceinline__ void join(const GqaArgs& a, int n, int id, ML m_of, O o_of, Partial<D>* part) {
  constexpr int kPerThread = kRows * D / kThreads;  // 8 or 4 consecutive dims of one row
  const int row = threadIdx.x / (D / kPerThread), d0 = (threadIdx.x % (D / kPerThread)) * kPerThread;
  const int grp = id % a.groups, kvh = id / a.groups % a.h_kv, b = id / a.groups / a.h_kv;
  const int r = grp * kRows + row;
  if (r >= a.g * a.s_q) return;
  float m = -INFINITY;
  for (int i = 0; i < n; ++i) m = fmaxf(m, m_of(i)[row]);
  float l = 0.f, o[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) o[k] = 0.f;
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float f = fast_exp2(m_of(i)[row] - base);  // 0 where nothing was seen
    l += f * m_of(i)[kRows + row];
    const float* v = o_of(i) + row * D + d0;
#pragma unroll
    for (int k = 0; k < kPerThread; k += 4) {
      const float4 x = *reinterpret_cast<const float4*>(v + k);
      o[k] += f * x.x;
      o[k + 1] += f * x.y;
      o[k + 2] += f * x.z;
      o[k + 3] += f * x.w;
    }
  }
  if (part) {
    if (d0 == 0) {
      part->m[row] = m;
      part->l[row] = l;
    }
#pragma unroll
    for (int k = 0; k < kPerThread; k += 4)
      *reinterpret_cast<float4*>(part->o + row * D + d0 + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
    return;
  }
  const bool none = m == -INFINITY;
  const float inv = none ? 0.f : 1.f / l;
  T* p = out_row<T>(a, b, kvh, r) + d0;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) o[k] *= inv;
  if constexpr (kPerThread == 8) {
    store_row16(p, o, 8);
  } else {
    uint2 w;
    if constexpr (std::is_same_v<T, __half>) {
      w = make_uint2(pack_half(o[0], o[1]), pack_half(o[2], o[3]));
    } else {
      const __nv_bfloat162 x = __floats2bfloat162_rn(o[0], o[1]), y = __floats2bfloat162_rn(o[2], o[3]);
      w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
    *reinterpret_cast<uint2*>(p) = w;
  }
  if (d0 == 0) *lse_at(a, b, kvh, r) = none ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
gqa_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const GqaArgs a) {
  using R = Ring<D, true>;
  constexpr int kStages = R::kStages;
  constexpr int kTiles = D / 8;  // n tiles of the output
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* first_o = reinterpret_cast<float*>(smem + kWarps * R::kBytes);  // [warp][16][D]
  DecodeShared<D>& sh = *reinterpret_cast<DecodeShared<D>*>(first_o + kWarps * kRows * D);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = lane >> 2, c = lane & 3;
  float* ring_o = reinterpret_cast<float*>(smem + warp * R::kBytes);
  const uint32_t ring = smem_u32(ring_o);
  uint64_t* full = sh.full[warp];

  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbarrier_init();
    sh.id[warp][0] = sh.id[warp][1] = -1;
  }
  if (tid == 0) sh.abort = 0;
  const int per_seq = a.h_kv * a.groups;
  const long long parts = (long long)gridDim.x * kWarps, first_part = (long long)blockIdx.x * kWarps;
  find_places(a, per_seq, kWarps, sh.list,
              [&](int k, long long total) { return piece_begin(total, first_part + k, parts); });
  const long long total = sh.list.total;
  long long left = piece_begin(total, first_part + warp + 1, parts) - piece_begin(total, first_part + warp, parts);
  const bool withhold = g_gqa_test_stall != 0 && tid == 0;

  // the two cursors: where loads and where products are
  struct Cursor {
    int b, kvh, grp, u, nu, len, end;  // end: the first query sees the positions below it
  };
  auto place = [&](Cursor& x, int b, long long u) {
    x.b = b;
    x.len = held_len(a, b);
    x.end = __ldg(a.ctx + b) - a.s_q + 1;
    x.nu = max(1, (x.len + kUnit - 1) / kUnit);
    const int pair = (int)(u / x.nu);
    x.u = (int)(u - (long long)pair * x.nu);
    x.kvh = pair / a.groups;
    x.grp = pair % a.groups;
  };
  auto advance = [&](Cursor& x) {
    if (++x.u < x.nu) return;
    x.u = 0;
    if (++x.grp < a.groups) return;
    x.grp = 0;
    if (++x.kvh < a.h_kv) return;
    x.kvh = 0;
    if (++x.b < a.b) {
      x.len = held_len(a, x.b);
      x.end = __ldg(a.ctx + x.b) - a.s_q + 1;
      x.nu = max(1, (x.len + kUnit - 1) / kUnit);
    }
  };
  Cursor ld = {}, cur = {};
  if (left > 0) {
    place(ld, sh.list.b[warp], sh.list.u[warp]);
    cur = ld;
  }
  long long to_load = left;
  Pages pages = {-1, -1, -1};
  float scales[kStages];
  int held[kStages];
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    scales[s] = 1.f;
    held[s] = 0;
    if (to_load > 0) {
      held[s] = load_unit<D, true>(a, &tk, &tv, pages, ld.b, ld.kvh, ld.u, ld.len, ring + s * R::kStage, &full[s],
                                   scales[s], withhold && s == 0);
      advance(ld);
      --to_load;
    }
  }

  uint32_t q[D / 16][4];
  float factor[2] = {0.f, 0.f};
  float o[kTiles][4], m[2], l[2], v_unit = 1.f;  // o is in units of v_unit
  int from = 0, slot = 0;
  bool fresh = true, ok = true;
  uint32_t phase = 0;
  const int rows = a.g * a.s_q;

  int st = 0;
  while (left > 0) {
    const int r0 = cur.grp * kRows;
    if (fresh) {
      load_q<T, D>(a, cur.b, cur.kvh, r0, rows, q, factor);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      v_unit = 1.f;
      from = cur.u;
      fresh = false;
    }
    const uint32_t k_stage = ring + st * R::kStage, v_stage = k_stage + R::kTile;
    // positions below `all` are seen by every row, those from `len` on by none
    const int t0 = cur.u * kUnit;
    const int all = min(cur.len, cur.end);
    int held_now = held[0];
    float scale_now = scales[0];
#pragma unroll
    for (int i = 1; i < kStages; ++i) {
      held_now = st == i ? held[i] : held_now;
      scale_now = st == i ? scales[i] : scale_now;
    }
    const float ks[2] = {__shfl_sync(0xffffffffu, scale_now, 0), __shfl_sync(0xffffffffu, scale_now, 1)};
    const float vs[2] = {__shfl_sync(0xffffffffu, scale_now, 2), __shfl_sync(0xffffffffu, scale_now, 3)};
    const bool edge = t0 + kUnit > all || held_now != 3 || vs[0] == 0.f || vs[1] == 0.f;
    const int lim[2] = {min(cur.len, cur.end + (r0 + j) / a.g), min(cur.len, cur.end + (r0 + j + 8) / a.g)};
    ok = mbar_wait(&full[st], phase, &sh.abort, &g_gqa_status);
    if (!ok) break;
    {
      float s[4][4];
      score_unit<D>(k_stage, q, s);
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = factor[i] * ks[nt >> 1];
          s[nt][2 * i] *= f;
          s[nt][2 * i + 1] *= f;
        }
      }
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          const bool there = (held_now >> (nt >> 1)) & 1;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int t = t0 + nt * 8 + Lay<D>::perm(2 * c + k);
            if (!there || t >= lim[0]) s[nt][k] = -INFINITY;
            if (!there || t >= lim[1]) s[nt][2 + k] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        top[0] = fmaxf(top[0], fmaxf(s[nt][0], s[nt][1]));
        top[1] = fmaxf(top[1], fmaxf(s[nt][2], s[nt][3]));
      }
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const float m_new = fmaxf(m[i], top[i]);
        alpha[i] = m_new == m[i] ? 1.f : fast_exp2(m[i] - m_new);
        m[i] = m_new;
        l[i] *= alpha[i];
      }
      const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[nt][2 * i] = fast_exp2(s[nt][2 * i] - base[i]);
          s[nt][2 * i + 1] = fast_exp2(s[nt][2 * i + 1] - base[i]);
          l[i] += s[nt][2 * i] + s[nt][2 * i + 1];
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {  // 16 positions each
        // o into units of these positions' v_scale (0: they add nothing)
        float r = 1.f;
        if ((held_now >> t) & 1) {
          if (vs[t] != 0.f && vs[t] != v_unit) {
            r = v_unit / vs[t];
            v_unit = vs[t];
          }
        }
        const float f0 = alpha[0] * r, f1 = alpha[1] * r;
        alpha[0] = alpha[1] = 1.f;
        if (!__all_sync(0xffffffffu, f0 == 1.f && f1 == 1.f)) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            o[i][0] *= f0;
            o[i][1] *= f0;
            o[i][2] *= f1;
            o[i][3] *= f1;
          }
        }
        const uint32_t p[4] = {pack_half(s[2 * t][0], s[2 * t][1]), pack_half(s[2 * t][2], s[2 * t][3]),
                               pack_half(s[2 * t + 1][0], s[2 * t + 1][1]),
                               pack_half(s[2 * t + 1][2], s[2 * t + 1][3])};
        // the four positions whose p this thread holds
        const int row[4] = {16 * t + Lay<D>::perm(2 * c), 16 * t + Lay<D>::perm(2 * c + 1),
                            16 * t + 8 + Lay<D>::perm(2 * c), 16 * t + 8 + Lay<D>::perm(2 * c + 1)};
        constexpr int kWords = kTiles / 4;  // 32-bit words per position
        uint32_t w[4][kWords];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (D == 128) {
            const uint4 x = lds_v4(v_stage + Lay<D>::piece(row[k], Lay<D>::col(j) / 16));
            w[k][0] = x.x;
            w[k][1] = x.y;
            w[k][2] = x.z;
            w[k][3] = x.w;
          } else {
            const uint2 x = lds_v2(v_stage + Lay<D>::piece(row[k], j >> 1) + (j & 1) * 8);
            w[k][0] = x.x;
            w[k][1] = x.y;
          }
        }
        // A position that some row does not see stays out of the
        // product: 0 * NaN of a stale or masked value would reach that
        // row.  Zero values here, added below for the rows that see them.
        if (edge) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool in = t0 + row[k] < all && ((held_now >> t) & 1) && vs[t] != 0.f;
#pragma unroll
            for (int e = 0; e < kWords; ++e) w[k][e] = in ? w[k][e] : 0u;
          }
        }
#pragma unroll
        for (int e = 0; e < kWords; ++e) {
          const uint32_t a01 = __byte_perm(w[0][e], w[1][e], 0x5140), a23 = __byte_perm(w[0][e], w[1][e], 0x7362);
          const uint32_t b01 = __byte_perm(w[2][e], w[3][e], 0x5140), b23 = __byte_perm(w[2][e], w[3][e], 0x7362);
          mma_f16(o[4 * e + 0], p, widen(a01 & 0xFFFFu), widen(b01 & 0xFFFFu));
          mma_f16(o[4 * e + 1], p, widen(a01 >> 16), widen(b01 >> 16));
          mma_f16(o[4 * e + 2], p, widen(a23 & 0xFFFFu), widen(b23 & 0xFFFFu));
          mma_f16(o[4 * e + 3], p, widen(a23 >> 16), widen(b23 >> 16));
        }
        if (edge && a.s_q > 1 && ((held_now >> t) & 1) && vs[t] != 0.f) {
          // the drafts' own positions: at most s_q - 1, row by row
          const int lo = max(max(all, 0), t0 + 16 * t), hi = min(cur.len, t0 + 16 * t + 16);
          for (int x = lo; x < hi; ++x) {
            const int in8 = (x - t0) & 7, half = ((x - t0) >> 3) & 1;
            const int col = Lay<D>::perm(in8);  // perm of Lay<64> is its own inverse
            const int cc = D == 128 ? ((in8 & 3) << 1 | (in8 >> 2)) : col;  // the column that holds position x
            const float x0 = half ? ((cc & 1) ? s[2 * t + 1][1] : s[2 * t + 1][0])
                                  : ((cc & 1) ? s[2 * t][1] : s[2 * t][0]);
            const float x1 = half ? ((cc & 1) ? s[2 * t + 1][3] : s[2 * t + 1][2])
                                  : ((cc & 1) ? s[2 * t][3] : s[2 * t][2]);
            const float p0 = __shfl_sync(0xffffffffu, x0, (lane & ~3) | (cc >> 1));
            const float p1 = __shfl_sync(0xffffffffu, x1, (lane & ~3) | (cc >> 1));
            const bool see0 = x < lim[0], see1 = x < lim[1];
            // this thread's columns: tile i, columns 2 c and 2 c + 1 are dims col(2 c) + i, col(2 c + 1) + i
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int dim = Lay<D>::col(2 * c + k) + i;
                uint32_t byte;
                asm volatile("ld.shared.u8 %0, [%1];"
                             : "=r"(byte)
                             : "r"(v_stage + Lay<D>::piece(x - t0, dim >> 4) + (dim & 15)));
                const uint32_t h2 = widen(byte);
                const float val = __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
                if (see0) o[i][k] += p0 * val;
                if (see1) o[i][2 + k] += p1 * val;
              }
            }
          }
        }
      }
      --left;
      const int now_u = cur.u, now_nu = cur.nu, now_b = cur.b, now_kvh = cur.kvh, now_grp = cur.grp;
      advance(cur);
      const bool done = now_u + 1 == now_nu;  // the (sequence, head, group) ends here
      __syncwarp();
      if (to_load > 0) {
        held_now = load_unit<D, true>(a, &tk, &tv, pages, ld.b, ld.kvh, ld.u, ld.len, k_stage, &full[st],
                                      scale_now, false);
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
          held[i] = st == i ? held_now : held[i];
          scales[i] = st == i ? scale_now : scales[i];
        }
        advance(ld);
        --to_load;
      }
      if (done || left == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        const bool whole = from == 0 && done;
        if (!whole && c == 0) {
          sh.m[warp][slot][j] = m[0];
          sh.m[warp][slot][j + 8] = m[1];
          sh.l[warp][slot][j] = l[0];
          sh.l[warp][slot][j + 8] = l[1];
        }
        if (!whole && lane == 0) {
          sh.id[warp][slot] = (now_b * a.h_kv + now_kvh) * a.groups + now_grp;
          sh.from[warp][slot] = from;
          sh.to[warp][slot] = now_u + 1;
          sh.nu[warp][slot] = now_nu;
        }
        float* keep = slot == 0 ? first_o + warp * kRows * D : ring_o;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + j + 8 * i;
          const float f = whole ? (m[i] == -INFINITY ? 0.f : v_unit / l[i]) : v_unit;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float v[kTiles];
#pragma unroll
            for (int e = 0; e < kTiles; ++e) v[e] = o[e][2 * i + k] * f;
            if (whole) {
              if (r < rows) store_row16(out_row<T>(a, now_b, now_kvh, r) + Lay<D>::col(2 * c + k), v, kTiles);
            } else {
#pragma unroll
              for (int e = 0; e < kTiles; e += 4)
                *reinterpret_cast<float4*>(keep + (j + 8 * i) * D + Lay<D>::col(2 * c + k) + e) =
                    make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
          }
          if (whole && c == 0 && r < rows)
            *lse_at(a, now_b, now_kvh, r) = m[i] == -INFINITY ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
        }
        if (!whole) slot = 1;
        fresh = true;
      }
    }
    if (++st == kStages) {
      st = 0;
      phase ^= 1;
    }
  }
  if (!ok) {  // this warp's loads in flight land (or their waits run out) before its shared memory goes
    const int flying = (int)min((long long)kStages, left - to_load);
    for (int i = 0; i < flying; ++i) {
      const int x = (st + i) % kStages;
      const long long t = clock64();
      while (!mbar_try_wait(smem_u32(&full[x]), phase ^ (x < st ? 1u : 0u), 1000u) && clock64() - t < kWaitLimitCycles) {
      }
    }
  }
  __syncthreads();

  // Pieces in order of the list: warp 0's first and last, warp 1's, ...
  Partial<D>* mine = reinterpret_cast<Partial<D>*>(a.ws) + (int64_t)blockIdx.x * 2;
  if (tid < 2) mine[tid].id = -1;
  __syncthreads();
  if (sh.abort) return;
  for (int x = 0; x < 2 * kWarps;) {
    const int id = sh.id[x >> 1][x & 1];
    if (id < 0) {
      ++x;
      continue;
    }
    int e = x + 1, last = x;
    while (e < 2 * kWarps && (sh.id[e >> 1][e & 1] == id || sh.id[e >> 1][e & 1] < 0)) {
      if (sh.id[e >> 1][e & 1] == id) last = e;
      ++e;
    }
    const bool begins = sh.from[x >> 1][x & 1] == 0;
    const bool ends = sh.to[last >> 1][last & 1] == sh.nu[last >> 1][last & 1];
    Partial<D>* part = begins && ends ? nullptr : mine + (begins ? 1 : 0);
    // the pieces x .. last that there are, as a dense list
    int idx[2 * kWarps], n = 0;
    for (int k = x; k <= last; ++k)
      if (sh.id[k >> 1][k & 1] == id) idx[n++] = k;
    __shared__ float ml[2 * kWarps][2 * kRows];
    for (int k = tid; k < n * kRows; k += kThreads) {
      const int p = idx[k / kRows];
      ml[k / kRows][k % kRows] = sh.m[p >> 1][p & 1][k % kRows];
      ml[k / kRows][kRows + k % kRows] = sh.l[p >> 1][p & 1][k % kRows];
    }
    __syncthreads();
    join<T, D>(a, n, id, [&](int i) -> const float* { return ml[i]; },
               [&](int i) -> const float* {
                 const int p = idx[i];
                 return (p & 1) ? reinterpret_cast<const float*>(smem + (p >> 1) * R::kBytes)
                                : first_o + (p >> 1) * kRows * D;
               },
               part);
    if (part && tid == 0) {
      part->id = id;
      part->begins = begins;
      part->ends = ends;
      // the CTA that holds the last unit of this (sequence, head, group)
      part->last = 0;
      if (!ends) {
        const long long here = piece_begin(total, first_part + (last >> 1) + 1, parts);  // list position after the piece
        const long long end = here + (sh.nu[last >> 1][last & 1] - sh.to[last >> 1][last & 1]);
        part->last = piece_of(total, end - 1, parts) / kWarps;
      }
    }
    __syncthreads();
    x = e;
  }
}

// Joins what several CTAs have of one (sequence, head, group): CTA i's, if
// it begins there.  The pieces lie in the CTAs up to `last` (a short list
// leaves some of them without a unit).
constexpr int kMaxCtas = 192;
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) gqa_join_kernel(const GqaArgs a) {
  __shared__ float ml[kMaxCtas][2 * kRows];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Partial<D>* all = reinterpret_cast<const Partial<D>*>(a.ws);
  const Partial<D>* p = all + (int64_t)blockIdx.x * 2 + 1;
  const int id = p->id;
  if (id < 0) return;
  const int n = p->last - (int)blockIdx.x + 1;
  auto piece = [&](int i) { return i == 0 ? p : all + (int64_t)(blockIdx.x + i) * 2; };
  for (int k = threadIdx.x; k < n * kRows; k += kThreads) {
    const Partial<D>* x = piece(k / kRows);
    const bool there = x->id == id;
    ml[k / kRows][k % kRows] = there ? x->m[k % kRows] : -INFINITY;
    ml[k / kRows][kRows + k % kRows] = there ? x->l[k % kRows] : 0.f;
  }
  __syncthreads();
  join<T, D>(a, n, id, [&](int i) -> const float* { return ml[i]; },
             // a piece that is not there has no values: any finite ones do, their factor is 0
             [&](int i) -> const float* { return ml[i][0] == -INFINITY && piece(i)->id != id ? p->o : piece(i)->o; },
             (Partial<D>*)nullptr);
}

// ------------------------------------------------------------------ weights
// One CTA takes a contiguous piece of the units of all (sequence, KV head)
// pairs, its warps every eighth unit of it.  A unit's 32 weights are the sum
// over all rows: thread (j, c) adds p of its rows, then the eight j are
// joined by a halving exchange that leaves one position per lane.  Rows of
// more than one group have their fragments of q in shared memory, up to
// kHeldGroups of them; more take further passes over the piece.
constexpr int kHeldGroups = 16;
template <int D>
struct WeightsShared {
  uint64_t full[kWarps][Ring<D, false>::kStages];
  ListShared list;
  float factor[kHeldGroups][kRows], lse[kHeldGroups][kRows];
  int abort;
};
template <int D, bool ONE>
constexpr int weights_smem() {
  return 1024 + kWarps * Ring<D, false>::kBytes + (ONE ? 0 : kHeldGroups * (D / 16) * 4 * 32 * 4) +
         (int)sizeof(WeightsShared<D>);
}

template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(kThreads, 1)
gqa_weights_kernel(const __grid_constant__ CUtensorMap tk, const GqaArgs a) {
  using R = Ring<D, false>;
  constexpr int kStages = R::kStages;
  constexpr int kQ = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* q_held = reinterpret_cast<uint4*>(smem + kWarps * R::kBytes);  // [group][k-step][lane]
  WeightsShared<D>& sh =
      *reinterpret_cast<WeightsShared<D>*>(smem + kWarps * R::kBytes + (ONE ? 0 : kHeldGroups * kQ * 32 * 16));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem + warp * R::kBytes);
  uint64_t* full = sh.full[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbarrier_init();
  }
  if (tid == 0) sh.abort = 0;
  const int rows = a.g * a.s_q;
  const long long parts = gridDim.x;
  find_places(a, a.h_kv, 1, sh.list, [&](int, long long total) { return piece_begin(total, blockIdx.x, parts); });
  const long long total = sh.list.total;
  const long long mine = piece_begin(total, blockIdx.x + 1, parts) - piece_begin(total, blockIdx.x, parts);
  const int b0 = sh.list.b[0];
  const long long u0 = mine > 0 ? sh.list.u[0] : 0;

  struct Cursor {
    int b, kvh, u, nu, len;
    long long left;
  };
  auto enter = [&](Cursor& x) {
    if (x.b >= a.b) return;
    x.len = held_len(a, x.b);
    x.nu = max(1, (x.len + kUnit - 1) / kUnit);
  };
  auto skip = [&](Cursor& x, int n) {  // n units on
    x.u += n;
    while (x.u >= x.nu && x.b < a.b) {
      x.u -= x.nu;
      if (++x.kvh == a.h_kv) {
        x.kvh = 0;
        ++x.b;
        enter(x);
      }
    }
  };
  Cursor start = {};
  if (mine > 0) {
    start.b = b0;
    enter(start);
    start.kvh = (int)(u0 / start.nu);
    start.u = (int)(u0 - (long long)start.kvh * start.nu);
  }
  const long long my_units = mine > warp ? (mine - warp + kWarps - 1) / kWarps : 0;
  Cursor first = start;  // this warp's first unit
  if (my_units > 0) skip(first, warp);
  first.left = my_units;

  uint32_t phase = 0;
  int st = 0;
  bool ok = true;
  uint32_t q[kQ][4];
  float factor[2], lse2[2];
  for (int g0 = 0; g0 < a.groups; g0 += kHeldGroups) {
    const int ng = min(kHeldGroups, a.groups - g0);
    Cursor ld = first, cur = first;
    Pages pages = {-1, -1, -1};
    float scales[kStages];
    int held[kStages];
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int x = (st + s) % kStages;
      float sc = 1.f;
      int h = 0;
      if (ld.left > 0 && ok) {
        h = load_unit<D, false>(a, &tk, &tk, pages, ld.b, ld.kvh, ld.u, ld.len, ring + x * R::kStage, &full[x], sc,
                                false);
        --ld.left;
        if (ld.left > 0) skip(ld, kWarps);
      }
#pragma unroll
      for (int i = 0; i < kStages; ++i) {
        held[i] = x == i ? h : held[i];
        scales[i] = x == i ? sc : scales[i];
      }
    }
    // the pairs of the piece, one after another
    Cursor pair = start;
    long long to_go = mine;
    bool fresh = true;
    while (to_go > 0) {
      const long long in_pair = min(to_go, (long long)(pair.nu - pair.u));
      if constexpr (!ONE) {
        __syncthreads();  // the last pair's fragments are read
        for (int gr = warp; gr < ng; gr += kWarps) {
          uint32_t f[kQ][4];
          float fac[2];
          load_q<T, D>(a, pair.b, pair.kvh, (g0 + gr) * kRows, rows, f, fac);
#pragma unroll
          for (int s = 0; s < kQ; ++s) q_held[(gr * kQ + s) * 32 + lane] = make_uint4(f[s][0], f[s][1], f[s][2], f[s][3]);
          if (c == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = (g0 + gr) * kRows + j + 8 * i;
              float e = INFINITY;  // a row that is not there, or saw nothing, adds exp2(-inf)
              if (r < rows) {
                e = __ldg(a.lse_in + ((int64_t)pair.b * a.h_q + pair.kvh * a.g + r % a.g) * a.s_q + r / a.g) * kLog2e;
                if (e == -INFINITY) e = INFINITY;
              }
              sh.factor[gr][j + 8 * i] = fac[i];
              sh.lse[gr][j + 8 * i] = e;
            }
          }
        }
        __syncthreads();
      }
      fresh = true;
      while (ok && cur.left > 0 && cur.b == pair.b && cur.kvh == pair.kvh) {
        if constexpr (ONE) {
          if (fresh) {
            load_q<T, D>(a, cur.b, cur.kvh, 0, rows, q, factor);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = j + 8 * i;
              lse2[i] = INFINITY;
              if (r < rows) {
                lse2[i] = __ldg(a.lse_in + ((int64_t)cur.b * a.h_q + cur.kvh * a.g + r % a.g) * a.s_q + r / a.g) * kLog2e;
                if (lse2[i] == -INFINITY) lse2[i] = INFINITY;
              }
            }
            fresh = false;
          }
        }
        int held_now = held[0];
        float scale_now = scales[0];
#pragma unroll
        for (int i = 1; i < kStages; ++i) {
          held_now = st == i ? held[i] : held_now;
          scale_now = st == i ? scales[i] : scale_now;
        }
        const float ks[2] = {__shfl_sync(0xffffffffu, scale_now, 0), __shfl_sync(0xffffffffu, scale_now, 1)};
        const int t0 = cur.u * kUnit;
        const int end = __ldg(a.ctx + cur.b) - a.s_q + 1;
        const bool edge = t0 + kUnit > min(cur.len, end) || held_now != 3;
        // the position whose weight this lane will hold
        const int t_mine = t0 + 8 * (j >> 1) + Lay<D>::perm(2 * c + (j & 1));
        float* w = a.weights + (int64_t)cur.b * a.stride_w_b + (int64_t)cur.kvh * a.stride_w_h + t_mine;
        const bool write = t_mine < cur.len && t_mine < a.width;
        const float before = write && (a.accumulate || g0 > 0) ? *w : 0.f;
        ok = mbar_wait(&full[st], phase, &sh.abort, &g_gqa_status);
        if (!ok) break;
        float sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.f;
        for (int gr = 0; gr < ng; ++gr) {
          if constexpr (!ONE) {
#pragma unroll
            for (int s = 0; s < kQ; ++s) {
              const uint4 f = q_held[(gr * kQ + s) * 32 + lane];
              q[s][0] = f.x;
              q[s][1] = f.y;
              q[s][2] = f.z;
              q[s][3] = f.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              factor[i] = sh.factor[gr][j + 8 * i];
              lse2[i] = sh.lse[gr][j + 8 * i];
            }
          }
          float s[4][4];
          score_unit<D>(ring + st * R::kStage, q, s);
          const int lim0 = end + ((g0 + gr) * kRows + j) / a.g, lim1 = end + ((g0 + gr) * kRows + j + 8) / a.g;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float p0 = fast_exp2(s[nt][k] * (factor[0] * ks[nt >> 1]) - lse2[0]);
              float p1 = fast_exp2(s[nt][2 + k] * (factor[1] * ks[nt >> 1]) - lse2[1]);
              if (edge) {
                const int t = t0 + nt * 8 + Lay<D>::perm(2 * c + k);
                const bool there = (held_now >> (nt >> 1)) & 1;
                p0 = there && t < lim0 ? p0 : 0.f;
                p1 = there && t < lim1 ? p1 : 0.f;
              }
              sum[2 * nt + k] += p0 + p1;
            }
          }
        }
        // eight values over the eight j: each step sends half of them
#pragma unroll
        for (int h = 4; h >= 1; h >>= 1) {
          const bool up = lane & (h * 4);
#pragma unroll
          for (int i = 0; i < h; ++i) {
            const float send = up ? sum[i] : sum[i + h], keep = up ? sum[i + h] : sum[i];
            sum[i] = keep + __shfl_xor_sync(0xffffffffu, send, h * 4);
          }
        }
        if (write) *w = before + sum[0];
        __syncwarp();
        if (ld.left > 0) {
          held_now = load_unit<D, false>(a, &tk, &tk, pages, ld.b, ld.kvh, ld.u, ld.len, ring + st * R::kStage,
                                         &full[st], scale_now, false);
#pragma unroll
          for (int i = 0; i < kStages; ++i) {
            held[i] = st == i ? held_now : held[i];
            scales[i] = st == i ? scale_now : scales[i];
          }
          --ld.left;
          if (ld.left > 0) skip(ld, kWarps);
        }
        --cur.left;
        if (cur.left > 0) skip(cur, kWarps);
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
      to_go -= in_pair;
      if (to_go > 0) skip(pair, (int)in_pair);
    }
    if (!ok) {  // this warp's loads in flight land (or their waits run out) before its shared memory goes
      const int flying = (int)min((long long)kStages, cur.left - ld.left);
      for (int i = 0; i < flying; ++i) {
        const int x = (st + i) % kStages;
        const long long t = clock64();
        while (!mbar_try_wait(smem_u32(&full[x]), phase ^ (x < st ? 1u : 0u), 1000u) &&
               clock64() - t < kWaitLimitCycles) {
        }
      }
      first.left = 0;
    }
  }
  if (!a.accumulate) {  // zeros behind each context
    for (int x = blockIdx.x; x < a.b * a.h_kv; x += gridDim.x) {
      float* w = a.weights + (int64_t)(x / a.h_kv) * a.stride_w_b + (int64_t)(x % a.h_kv) * a.stride_w_h;
      for (int t = held_len(a, x / a.h_kv) + tid; t < a.width; t += kThreads) w[t] = 0.f;
    }
  }
}

// ------------------------------------------------------------------ host
// [num_blocks][h_kv][page][d] of one byte, boxes of up to 32 rows of a head.
bool make_map(CUtensorMap* m, const void* base, int64_t stride_block, int64_t stride_row, int64_t stride_head,
              const dsv4b_gqa_cache& c) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c.d, (cuuint64_t)c.page_block_size, (cuuint64_t)c.h_kv,
                              (cuuint64_t)c.num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)stride_row, (cuuint64_t)stride_head, (cuuint64_t)stride_block};
  const cuuint32_t box[4] = {(cuuint32_t)c.d, (cuuint32_t)(c.page_block_size < kUnit ? c.page_block_size : kUnit), 1, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, c.d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

GqaArgs make_args(const dsv4b_gqa_cache& c, const dsv4b_gqa_query& q) {
  GqaArgs a = {};
  a.q = q.q;
  a.stride_q_b = q.stride_q_b;
  a.stride_q_s = q.stride_q_s;
  a.stride_q_h = q.stride_q_h;
  a.s_q = q.s_q;
  a.h_q = q.h_q;
  a.h_kv = c.h_kv;
  a.g = q.h_q / c.h_kv;
  a.groups = (a.g * q.s_q + kRows - 1) / kRows;
  a.scale_log2 = q.sm_scale * kLog2e;
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  a.table = c.block_table;
  a.stride_table = c.stride_block_table;
  a.table_width = c.table_width;
  a.num_blocks = c.num_blocks;
  a.page = c.page_block_size;
  while ((1 << a.page_shift) < a.page) ++a.page_shift;
  a.b = c.b;
  a.ctx = c.context_lens;
  return a;
}

int grid_of(int sms) { return sms < kMaxCtas ? sms : kMaxCtas; }

template <typename K>
cudaError_t allow_smem(K* kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

template <typename T, int D>
cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const GqaArgs& a, int grid,
                          cudaStream_t stream) {
  constexpr int smem = decode_smem<D>();
  static_assert(smem <= 227 * 1024, "decode kernel shared memory");
  static bool done[64] = {};
  cudaError_t e = allow_smem(&gqa_decode_kernel<T, D>, smem, done);
  if (e != cudaSuccess) return e;
  gqa_decode_kernel<T, D><<<grid, kThreads, smem, stream>>>(tk, tv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;  // its launch overlaps the decode; it waits in the kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, gqa_join_kernel<T, D>, a);
}

template <typename T, int D, bool ONE>
cudaError_t launch_weights(const CUtensorMap& tk, const GqaArgs& a, int grid, cudaStream_t stream) {
  constexpr int smem = weights_smem<D, ONE>();
  static_assert(smem <= 227 * 1024, "weights kernel shared memory");
  static bool done[64] = {};
  cudaError_t e = allow_smem(&gqa_weights_kernel<T, D, ONE>, smem, done);
  if (e != cudaSuccess) return e;
  gqa_weights_kernel<T, D, ONE><<<grid, kThreads, smem, stream>>>(tk, a);
  return cudaGetLastError();
}

}  // namespace

size_t gqa_decode_ws_bytes(int sms, int d) {
  return (size_t)grid_of(sms) * 2 * (d == 128 ? sizeof(Partial<128>) : sizeof(Partial<64>));
}

cudaError_t launch_gqa_decode(const dsv4b_gqa_cache& c, const dsv4b_gqa_query& q, void* out, int64_t stride_o_b,
                              int64_t stride_o_s, int64_t stride_o_h, float* lse, void* ws, int sms,
                              cudaStream_t stream, int* bad_arg) {
  CUtensorMap tk, tv;
  if (!make_map(&tk, c.k, c.stride_k_block, c.stride_k_row, c.stride_k_head, c) ||
      !make_map(&tv, c.v, c.stride_v_block, c.stride_v_row, c.stride_v_head, c)) {
    *bad_arg = 1;
    return cudaErrorInvalidValue;
  }
  GqaArgs a = make_args(c, q);
  a.out = out;
  a.stride_o_b = stride_o_b;
  a.stride_o_s = stride_o_s;
  a.stride_o_h = stride_o_h;
  a.lse = lse;
  a.ws = static_cast<float*>(ws);
  const int grid = grid_of(sms);
  if (q.dtype == DSV4B_BF16)
    return c.d == 128 ? launch_decode<__nv_bfloat16, 128>(tk, tv, a, grid, stream)
                      : launch_decode<__nv_bfloat16, 64>(tk, tv, a, grid, stream);
  return c.d == 128 ? launch_decode<__half, 128>(tk, tv, a, grid, stream)
                    : launch_decode<__half, 64>(tk, tv, a, grid, stream);
}

cudaError_t launch_gqa_weights(const dsv4b_gqa_cache& c, const dsv4b_gqa_query& q, const float* lse, float* weights,
                               int64_t stride_w_b, int64_t stride_w_h, int width, int accumulate, int sms,
                               cudaStream_t stream, int* bad_arg) {
  CUtensorMap tk;
  if (!make_map(&tk, c.k, c.stride_k_block, c.stride_k_row, c.stride_k_head, c)) {
    *bad_arg = 1;
    return cudaErrorInvalidValue;
  }
  GqaArgs a = make_args(c, q);
  a.lse_in = lse;
  a.weights = weights;
  a.stride_w_b = stride_w_b;
  a.stride_w_h = stride_w_h;
  a.width = width;
  a.accumulate = accumulate;
  const int grid = grid_of(sms);
  const bool one = a.groups == 1;  // one group's q stays in registers, without a barrier per pair
  if (q.dtype == DSV4B_BF16) {
    if (c.d == 128)
      return one ? launch_weights<__nv_bfloat16, 128, true>(tk, a, grid, stream)
                 : launch_weights<__nv_bfloat16, 128, false>(tk, a, grid, stream);
    return one ? launch_weights<__nv_bfloat16, 64, true>(tk, a, grid, stream)
               : launch_weights<__nv_bfloat16, 64, false>(tk, a, grid, stream);
  }
  if (c.d == 128)
    return one ? launch_weights<__half, 128, true>(tk, a, grid, stream)
               : launch_weights<__half, 128, false>(tk, a, grid, stream);
  return one ? launch_weights<__half, 64, true>(tk, a, grid, stream)
             : launch_weights<__half, 64, false>(tk, a, grid, stream);
}

cudaError_t read_gqa_status(int* flags, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(flags, g_gqa_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return e;
  if ((e = cudaStreamSynchronize(stream)) != cudaSuccess) return e;
  static const int zero = 0;
  return cudaMemcpyToSymbolAsync(g_gqa_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
}

cudaError_t set_gqa_test_stall(int stall) { return cudaMemcpyToSymbol(g_gqa_test_stall, &stall, sizeof(stall)); }

}  // namespace dsv4b
