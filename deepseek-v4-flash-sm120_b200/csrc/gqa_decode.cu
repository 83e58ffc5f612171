// Attention over the 8-bit grouped-query cache, and the attention weights of
// its positions (include/dsv4b.h, dsv4b_gqa_decode and
// dsv4b_gqa_attention_weights).
//
//   s[r][t] = sm_scale * k_scale * sum_d q[r][d] * k[t][d]
//   out[r]  = sum_t exp(s[r][t] - lse[r]) * v_scale * v[t]
// for the rows r = (query, head) that share a KV head: h_q / h_kv * s_q of
// them, in decode few against the positions.  Every cached byte is used for
// all rows (of a group of 8 or 16) at once and only once, so decode and the
// weights of few rows are bound by the cache's bytes.
//
// Work.  A unit is 64 positions of one (sequence, KV head, group of 8 or 16
// rows).  All units stand in one list, and every warp of the grid (one CTA
// per SM) takes an equal, contiguous piece of it, so ragged batches balance
// without a plan made ahead.  A warp runs the softmax of its piece by
// itself: no barrier until its CTA's end, where pieces of one (sequence,
// head, group) are joined; those that reach over CTAs are joined by a second
// kernel.
//
// Loads.  Each warp has its own ring of 64-position tiles, K and V in turn
// (8 KB each at d = 128), filled by TMA tiled loads that swizzle the rows
// and counted on mbarriers: up to 192 KB are in flight on an SM, without a
// register or an issue slot spent on them.
//
// Measured, d = 128, against 6.5 TB/s of a copy: 16 sequences of 131,072
// positions, 8 KV heads of 16 rows (4.1 GB) 728 us, 5.6 TB/s (855 where it runs
// for long, at the power limit's 1.7 GHz); 32 of 1,000 to 32,768 with 8 rows
// (554 MB) 126 us, 4.4 TB/s; one of 4,096 (8.4 MB) 16.6.  The last is what a
// call takes whatever its size (launch, the list, the first tiles behind their
// page ids, the joins), of which the middle one shows about 14 us; for the rest
// its warps wait on memory for 40 % of their time and at barriers for 4 %.
//
// Products.  mma.sync m16n8k16 with fp16 operands, positions (or dims of V)
// as M and rows as N = 8: s^T = k q^T, out^T = v^T p^T.  The operands of
// tcgen05 would have to stand in shared memory in their final type, so e4m3
// would be widened into shared memory (twice its bytes written and read
// again) for a tile of which 8 rows are used; mma.sync takes them from
// registers, where an e4m3 pair becomes an fp16 pair (exactly) in one
// instruction, and its rate (974 multiply-adds a cycle and SM, measured) is
// above what the loads can feed.  The order of d in q.k and of the positions
// in p.v is free, so the fragments are built from 16-byte pieces of whole
// rows, thread (g, c) = (lane / 4, lane % 4):
//   K: it reads bytes [16c, 16c + 16) (and 64 further) of the positions
//      perm(g) and 8 + perm(g): four k-steps, with q laid out to match;
//   V: it reads the 16 dims from col(g) on of the four positions perm(2c),
//      perm(2c + 1) and 8 further, and interleaves the bytes of two.
// perm and col make every such read free of bank conflicts (below).  s^T
// has a position per g and rows 2c, 2c + 1 in a thread; transposing its 8x8
// blocks (movmatrix) gives p^T's fragments.
//
// Numbers.  q is scaled by a power of two per row so that fp16 holds it
// (bf16 has fewer digits; what lies 2^-27 below the row's largest loses some,
// 2^-37 below it all).
// p is relative to m, which lies 2^7 below the running maximum and is moved
// only when a score outgrows that by 2^8, so p <= 2^15: fp16's range is used
// up to its end, for the small p of a long context (2^-14 of the maximum and
// less would lose digits, 2^-25 be gone with m at the maximum).  p is rounded
// to fp16 for p.v (2^-11 of each term, 2^-32 of the maximum at least), sums and
// the softmax's denominator are fp32 of the unrounded p.  The accumulator is
// kept in units of the current block's v_scale and rescaled when that or m
// changes, so that no scale enters an fp16.  A v_scale may be anything (append
// gives a block of zeros 2^-100), so the unit stays within 2^64 of the
// largest so far: sums of 2^30 positions keep below 2^119 units, and go up to
// any larger unit by factors of 2^-100 at least.  Blocks further down leave
// the unit and are added position by position, in fp32, if they hold anything
// but zeros.  A piece's values are kept divided by their sum, as large as V.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "dsv4b.h"
#include "dsv4b_kernels.h"
#include "dsv4b_ptx.cuh"
#include "gqa_tc.cuh"

namespace dsv4b {

__device__ int g_gqa_status;  // kErr* bits of the grouped-query kernels on this device
// Test hook (dsv4b_set_test_stall): when set, the first load of every CTA
// is withheld, so that the first wait runs out.
__device__ int g_gqa_test_stall = 0;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBelow = 7.f;    // log2 of how far m is put below the largest score
constexpr float kRescale = 8.f;  // log2 of how far that may be outgrown: p <= 2^15
constexpr float kUnitSpan = 5.421010862427522e-20f;  // 2^-64: the least unit of o beside the largest v_scale

struct GqaArgs {
  const void* q;
  int64_t stride_q_b, stride_q_s, stride_q_h;
  int s_q, h_q, h_kv, g, groups;  // g = h_q / h_kv; groups of rows per KV head
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

// Positions of sequence i that the call reads.
__device__ __forceinline__ int held_len(const GqaArgs& a, int i) {
  const int64_t room = (int64_t)a.table_width * a.page;
  return (int)min((int64_t)max(__ldg(a.ctx + i), 0), room);
}
// Its units of U positions (one at least: an empty sequence has its outputs written too).
template <int U>
__device__ __forceinline__ int units_of(int len) {
  return max(1, (len + U - 1) / U);
}

// ------------------------------------------------------------------ layouts
// Rows of d bytes, swizzled by TMA: 16-byte piece p of row r lies at
// p ^ (r & 7) (128-byte rows) or p ^ ((r >> 1) & 3) (64-byte rows).
template <int D>
struct Lay;
template <>
struct Lay<128> {
  // A quarter of a warp's 16-byte reads (8 threads) is g, g + 1 with all c,
  // for K and for V.  Rows that differ in bit 2 swap the halves of the row,
  // so K wants perm(2i), perm(2i + 1) four apart and V wants col(2i),
  // col(2i + 1) four pieces apart.
  static __device__ __forceinline__ int perm(int i) { return (i >> 1) | ((i & 1) << 2); }
  static __device__ __forceinline__ int unperm(int t) { return ((t & 3) << 1) | (t >> 2); }
  static __device__ __forceinline__ int col(int i) { return ((i >> 1) | ((i & 1) << 2)) * 16; }  // dims [col, col + 16)
  static __device__ __forceinline__ uint32_t piece(int row, int p) { return row * 128 + ((p ^ (row & 7)) << 4); }
};
template <>
struct Lay<64> {
  // Two rows share 128 bytes, the odd one in the upper half: K wants
  // perm(2i), perm(2i + 1) of different parity, V (8-byte reads, 16 threads
  // at once) wants perm(0), perm(2), perm(4), perm(6) of changing parity.
  static __device__ __forceinline__ int perm(int i) { return i ^ ((i >> 1) & 1); }
  static __device__ __forceinline__ int unperm(int t) { return t ^ ((t >> 1) & 1); }
  static __device__ __forceinline__ int col(int i) { return i * 8; }  // dims [col, col + 8)
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
// The D / 8 bytes of V's dims from col(g) on, of one row of a tile.
template <int D>
__device__ __forceinline__ void lds_v_row(uint32_t tile, int row, int g, uint32_t (&w)[D / 32]) {
  if constexpr (D == 128) {
    const uint4 x = lds_v4(tile + Lay<D>::piece(row, Lay<D>::col(g) / 16));
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  } else {
    const uint2 x = lds_v2(tile + Lay<D>::piece(row, g >> 1) + (g & 1) * 8);
    w[0] = x.x;
    w[1] = x.y;
  }
}

// Two e4m3 (low byte first) as two fp16, exactly.
__device__ __forceinline__ uint32_t widen(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The two pairs of a word.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8x8 block of 16-bit values (row g, columns 2c, 2c + 1 in a thread), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Four 16-bit values.
template <typename T>
__device__ __forceinline__ float4 four(uint2 w) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
  }
}

// The largest magnitude of eight 16-bit values, as the bits of an fp32 (NaN counts as more).
template <typename T>
__device__ __forceinline__ uint32_t largest(uint4 w) {
  const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
  const uint32_t top = max(m & 0xFFFFu, m >> 16);
  if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  return top << 16;
}

// The q^T fragments of 8 rows from row r0 on: thread (g, c) holds row g, for
// k-step 4 h + s the dims 16 (4 h + c) + 4 s + {0, 1, 2, 3}, the same that
// it reads of K.  Rows from `rows` on are zero.  factor[k] is what the
// products of row 2c + k are multiplied by: the row's power of two and the
// softmax scale.
template <int D>
struct RawQ {
  uint2 w[D / 16];
};
template <typename T, int D>
__device__ __forceinline__ void fetch_q(const GqaArgs& a, int b, int kvh, int r0, int rows, RawQ<D>& raw) {
  const int lane = threadIdx.x & 31, c = lane & 3, r = r0 + (lane >> 2);
  const bool live = r < rows;
  const T* p = static_cast<const T*>(a.q);
  if (live)
    p += (int64_t)b * a.stride_q_b + (int64_t)(r / a.g) * a.stride_q_s + (int64_t)(kvh * a.g + r % a.g) * a.stride_q_h;
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
    raw.w[s] = live ? __ldg(reinterpret_cast<const uint2*>(p + (s >> 2) * 64 + c * 16 + (s & 3) * 4)) : make_uint2(0, 0);
}
// A row of q's power of two (its largest value `top` becomes 2^13 .. 2^14; an
// infinite one stays so), and what its products are multiplied by.
__device__ __forceinline__ void row_scale(const GqaArgs& a, float top, float& up, float& down) {
  const int e = min(max((int)(__float_as_uint(top) >> 23), 40), 254) - 127 - 13;
  up = __uint_as_float((uint32_t)(127 - e) << 23);
  down = a.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23);
}
template <typename T, int D>
__device__ __forceinline__ void scale_q(const GqaArgs& a, const RawQ<D>& raw, uint32_t (&q)[D / 16][2],
                                        float (&factor)[2]) {
  const int c = threadIdx.x & 3;
  float4 f[D / 16];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    f[s] = four<T>(raw.w[s]);
    top = fmaxf(top, fmaxf(fmaxf(fabsf(f[s].x), fabsf(f[s].y)), fmaxf(fabsf(f[s].z), fabsf(f[s].w))));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  float up, down;
  row_scale(a, top, up, down);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    q[s][0] = pack_half(f[s].x * up, f[s].y * up);
    q[s][1] = pack_half(f[s].z * up, f[s].w * up);
  }
  factor[0] = __shfl_sync(0xffffffffu, down, 8 * c);
  factor[1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
}
template <typename T, int D>
__device__ __forceinline__ void load_q(const GqaArgs& a, int b, int kvh, int r0, int rows, uint32_t (&q)[D / 16][2],
                                       float (&factor)[2]) {
  RawQ<D> raw;
  fetch_q<T, D>(a, b, kvh, r0, rows, raw);
  scale_q<T, D>(a, raw, q, factor);
}

// K's fragments of 16 positions of a tile for k-steps 4 h .. 4 h + 3.
template <int D>
__device__ __forceinline__ void k_frags(uint32_t tile, int mt, int h, uint32_t (&f)[4][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint4 x = lds_v4(tile + Lay<D>::piece(mt * 16 + Lay<D>::perm(g), 4 * h + c));
  const uint4 y = lds_v4(tile + Lay<D>::piece(mt * 16 + 8 + Lay<D>::perm(g), 4 * h + c));
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    widen4(xs[s], f[s][0], f[s][2]);
    widen4(ys[s], f[s][1], f[s][3]);
  }
}

// ------------------------------------------------------------------ the list
// `parts` equal pieces of a list (the first `more` of them one unit longer):
// where piece i begins, and which piece holds position x.
struct Split {
  long long each;
  int more;
  __device__ __forceinline__ Split(long long total, int parts) {
    if (total < (1ll << 31)) {  // a 64-bit division takes a microsecond of a cold start
      each = (unsigned)total / (unsigned)parts;
      more = (int)((unsigned)total - (unsigned)each * (unsigned)parts);
    } else {
      each = total / parts;
      more = (int)(total - each * parts);
    }
  }
  __device__ __forceinline__ long long begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int holder(long long x) const {
    const long long longer = (each + 1) * more;
    return x < longer ? (int)(x / (each + 1)) : more + (int)((x - longer) / each);
  }
};

template <int W>
struct ListShared {
  long long sum[W], pre[W * 32];
  long long total;
  int b[W];
  long long u[W];
};

// Where n pieces, from part0 on, of `parts` equal ones of the list of all
// sequences' units (per_seq times over for a sequence's heads and groups)
// begin: sh.b[k] the sequence (-1: past the end), sh.u[k] the unit among all
// of the sequence's.  Every thread sums a run of sequences, the sums are
// scanned, and a thread per piece searches the scan and walks the run that
// holds its beginning (the run's own thread, for all pieces in it, took 2,000
// cycles more where one sequence holds them all).
template <int W, int U>
__device__ __forceinline__ void find_places(const GqaArgs& a, int per_seq, int part0, int n, int parts,
                                            ListShared<W>& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (a.b + W * 32 - 1) / (W * 32);
  const int i0 = min(a.b, tid * run), i1 = min(a.b, i0 + run);
  long long sum = 0;
  for (int i = i0; i < i1; ++i) sum += units_of<U>(held_len(a, i));
  sum *= per_seq;
  long long incl = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.sum[warp] = incl;
  __syncthreads();
  long long pre = incl - sum, total = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < warp) pre += sh.sum[i];
    total += sh.sum[i];
  }
  if (tid == 0) sh.total = total;
  sh.pre[tid] = pre;
  __syncthreads();
  if (tid < n) {
    const long long x = Split(total, parts).begin(part0 + tid);
    sh.b[tid] = -1;
    if (x < total) {
      int j = 0;  // the last run that begins at or before x (an empty one begins where the next does)
#pragma unroll 1
      for (int o = 512; o; o >>= 1)
        if (j + o < W * 32 && sh.pre[j + o] <= x) j += o;
      long long at = sh.pre[j];
      for (int i = j * run; i < a.b; ++i) {
        const long long m = (long long)units_of<U>(held_len(a, i)) * per_seq;
        if (x < at + m) {
          sh.b[tid] = i;
          sh.u[tid] = x - at;
          break;
        }
        at += m;
      }
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------ loading
// The blocks of 512 positions of a (sequence, KV head), one per 16 of them,
// in the lanes: ids and scales (a load per unit would have its latency waited
// for in every unit).  `base` is the first unit's number (-1: none held).
struct Pages {
  int id, base, b, kvh;
  float ks, vs;
};
template <int U, bool WITH_V>
__device__ __forceinline__ void fetch_pages(const GqaArgs& a, Pages& p, int b, int kvh, int u, int len) {
  constexpr int kUnits = 512 / U;
  if (p.base == (u & ~(kUnits - 1)) && p.b == b && p.kvh == kvh) return;
  const int lane = threadIdx.x & 31;
  p.b = b;
  p.kvh = kvh;
  p.base = u & ~(kUnits - 1);
  const long long t = (long long)p.base * U + lane * 16;
  p.id = -1;
  p.ks = p.vs = 1.f;
  if (t < len) {
    const int id = __ldg(a.table + (int64_t)b * a.stride_table + (int)(t >> a.page_shift));
    if (id >= 0 && id < a.num_blocks) {
      p.id = id;
      p.ks = __ldg(a.k_scale + (int64_t)id * a.h_kv + kvh);
      if constexpr (WITH_V) p.vs = __ldg(a.v_scale + (int64_t)id * a.h_kv + kvh);
    }
  }
}

// What is known of a unit: which of its runs of 16 positions are there (one
// bit each), and the scales of their K and V.
template <int U>
struct Info {
  int held;
  float ks[U / 16], vs[U / 16];
};

// A tile of U positions in a warp's ring: K's or V's of unit u.  The maps'
// boxes have min(page, 64) rows (or 32, where U is); `ids` are the blocks of
// its runs of 16 (< 0: not there, not loaded).  One lane's work.
template <int D, int U>
__device__ __forceinline__ void load_tile(const GqaArgs& a, const CUtensorMap* map, const int (&ids)[U / 16], int kvh,
                                          int u, uint32_t tile, uint64_t* bar) {
  constexpr int kBytes = U * D;
  if (a.page >= U) {  // one block holds the unit (its last runs too, read or not)
    mbar_arrive_expect_tx(bar, ids[0] >= 0 ? kBytes : 0);
    if (ids[0] >= 0) tma_load_4d(tile, map, 0, (u * U) & (a.page - 1), kvh, ids[0], bar);
  } else {
    const int runs = a.page >> 4;  // of a block: 1, 2 or 4
    int n = 0;
#pragma unroll
    for (int i = 0; i < U / 16; ++i) n += ((i & (runs - 1)) == 0 && ids[i] >= 0) ? 1 : 0;
    mbar_arrive_expect_tx(bar, n * a.page * D);
#pragma unroll
    for (int i = 0; i < U / 16; ++i)
      if ((i & (runs - 1)) == 0 && ids[i] >= 0) tma_load_4d(tile + i * 16 * D, map, 0, 0, kvh, ids[i], bar);
  }
}

// After a wait gave up: a warp's loads in flight land (or their waits run
// out) before its shared memory goes.
__device__ __forceinline__ void drain(uint64_t* full, int slots, int slot, uint32_t phase, int flying) {
  for (int i = 0; i < slots && i < flying; ++i) {
    const int x = (slot + i) % slots;
    const long long t = clock64();
    while (!mbar_try_wait(smem_u32(&full[x]), phase ^ (x < slot ? 1u : 0u), 1000u) && clock64() - t < kWaitLimitCycles) {
    }
  }
}

// ------------------------------------------------------------------ decode
// A unit is 64 positions: what a unit costs beside its products (waits, the
// cursors, page ids, the loads' issue) is about 250 instructions of a warp,
// which at 32 positions took more issue slots than the products.  Up to 8
// rows of a head (one n-tile) leave room for 12 warps of 168 registers, 16
// rows for 8 of 255.
template <int D, int NT>
struct Dec {
  static constexpr int kUnit = 64;
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * NT;
  static constexpr int kTile = kUnit * D;
  static constexpr int kSlots = NT == 1 && D == 128 ? 2 : 3;
};

// A piece of one (sequence, head, group of rows): id numbers these; last:
// the CTA that holds its last unit.  o is divided by l, which is relative to
// 2^m.
template <int D, int NT>
struct Partial {
  int id, last, unused[2];
  float m[8 * NT], l[8 * NT];
  float o[8 * NT * D];
};
// Workspace: the CTAs' joined pieces ([CTA][2]: one whose beginning lies in
// an earlier CTA, one that goes on in the next), then the values of warps'
// first pieces ([CTA][warp][rows][D]).
template <int D, int NT>
constexpr size_t ws_bytes(int ctas) {
  return (size_t)ctas * (2 * sizeof(Partial<D, NT>) + (size_t)Dec<D, NT>::kWarps * 8 * NT * D * 4);
}

template <int D, int NT>
struct DecodeShared {
  using C = Dec<D, NT>;
  uint64_t full[C::kWarps][C::kSlots];
  ListShared<C::kWarps> list;
  // The pieces that a warp began ([0]) and ended ([1]) with, where they are
  // not whole.  Values of one that a warp ends with lie in its ring, which
  // it no longer needs; others in the workspace.
  int id[2 * C::kWarps];  // -1: none
  int from[2 * C::kWarps], to[2 * C::kWarps], nu[2 * C::kWarps], in_ring[2 * C::kWarps];
  float ml[2 * C::kWarps][2 * C::kRows];  // m, l
  // A warp's unit of o (0: o holds nothing), and the least one that it may
  // take: kUnitSpan times the largest v_scale so far.  Here for want of registers.
  float unit[C::kWarps], least_unit[C::kWarps];
  int list_of[2 * C::kWarps], run[2 * C::kWarps + 1], n_runs;
  int abort;
};
template <int D, int NT>
constexpr int decode_smem() {
  using C = Dec<D, NT>;
  return 1024 + C::kWarps * C::kSlots * C::kTile + (int)sizeof(DecodeShared<D, NT>);
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    return pack_half(lo, hi);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
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

constexpr int kMaxCtas = 192;

// Joins n pieces of one (sequence, head, group), in order, for the four
// consecutive values from e on of its [rows][D]: piece i has maxima and sums
// ml_of(i) (m, then l) and values o_of(i).  Writes the result, or the joined
// piece to `part`.
template <typename T, int D, int NT, typename ML, typename O>
__device__ __forceinline__ void join(const GqaArgs& a, int e, int n, int id, ML ml_of, O o_of, Partial<D, NT>* part) {
  constexpr int kRows = 8 * NT;
  const int grp = id % a.groups, kvh = id / a.groups % a.h_kv, b = id / a.groups / a.h_kv;
  const int row = e / D, d0 = e % D;
  const int r = grp * kRows + row;
  if (r >= a.g * a.s_q) return;
  float m = -INFINITY, most = 0.f;
  for (int i = 0; i < n; ++i) {
    m = fmaxf(m, ml_of(i)[row]);
    most = fmaxf(most, ml_of(i)[kRows + row]);
  }
  const float base = m == -INFINITY ? 0.f : m;
  // Sums of up to 192 pieces that weigh 2^-8 at most are no larger than V (a
  // power of two: no division).
  const float scale = __uint_as_float((254u << 23) - (__float_as_uint(most) & 0x7F800000u)) * 0x1p-9f;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kDeep = 8;  // loads in flight
  for (int i0 = 0; i0 < n; i0 += kDeep) {
    float4 x[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) x[i] = *reinterpret_cast<const float4*>(o_of(min(i0 + i, n - 1)) + e);
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      if (i0 + i < n) {
        const float w = fast_exp2(ml_of(i0 + i)[row] - base) * ml_of(i0 + i)[kRows + row];  // 0 where nothing was seen
        const float f = w * scale;
        l += w;
        o.x += f * x[i].x;
        o.y += f * x[i].y;
        o.z += f * x[i].z;
        o.w += f * x[i].w;
      }
    }
  }
  const bool none = l == 0.f;  // (not by m: a row of NaN scores has none, and is NaN)
  const float inv = none ? 0.f : 1.f / (l * scale);
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (part) {
    if (d0 == 0) {
      part->m[row] = m;
      part->l[row] = l;
    }
    *reinterpret_cast<float4*>(part->o + e) = o;
    return;
  }
  *reinterpret_cast<uint2*>(out_row<T>(a, b, kvh, r) + d0) = make_uint2(pack16<T>(o.x, o.y), pack16<T>(o.z, o.w));
  if (d0 == 0) *lse_at(a, b, kvh, r) = none ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Dec<D, NT>::kThreads, 1)
gqa_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const GqaArgs a) {
  using C = Dec<D, NT>;
  constexpr int kWarps = C::kWarps, kSlots = C::kSlots, kRows = C::kRows, kTile = C::kTile;
  constexpr int kUnit = C::kUnit, kRuns = kUnit / 16;
  constexpr int kSteps = D / 16;  // k-steps of q.k, m-tiles of the output
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  DecodeShared<D, NT>& sh = *reinterpret_cast<DecodeShared<D, NT>*>(smem + kWarps * kSlots * kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem + warp * kSlots * kTile);
  uint64_t* full = sh.full[warp];
  // in the workspace: the values of a warp's first piece
  auto first_o = [&](int w) {
    return reinterpret_cast<float*>(reinterpret_cast<Partial<D, NT>*>(a.ws) + (int64_t)gridDim.x * 2) +
           ((int64_t)blockIdx.x * kWarps + w) * kRows * D;
  };

  if (lane == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(&full[s], 1);
    fence_mbarrier_init();
    sh.id[2 * warp] = sh.id[2 * warp + 1] = -1;
  }
  if (tid == 0) sh.abort = 0;
  const int parts = gridDim.x * kWarps, first_part = blockIdx.x * kWarps;
  find_places<kWarps, kUnit>(a, a.h_kv * a.groups, first_part, kWarps, parts, sh.list);
  const Split split(sh.list.total, parts);
  int left = (int)split.each + (first_part + warp < split.more ? 1 : 0);

  // the two cursors: where loads and where products are
  struct Cursor {
    int b, kvh, grp, u, nu, len, end;  // end: the first query sees the positions below it
  };
  auto enter = [&](Cursor& x) {
    x.len = held_len(a, x.b);
    x.end = __ldg(a.ctx + x.b) - a.s_q + 1;
    x.nu = units_of<kUnit>(x.len);
  };
  auto advance = [&](Cursor& x) {
    if (++x.u < x.nu) return;
    x.u = 0;
    if (++x.grp < a.groups) return;
    x.grp = 0;
    if (++x.kvh < a.h_kv) return;
    x.kvh = 0;
    if (++x.b < a.b) enter(x);
  };
  Cursor cur = {};
  if (left > 0) {
    cur.b = sh.list.b[warp];
    enter(cur);
    const long long u = sh.list.u[warp];
    const int pair = u < (1ll << 31) ? (int)((unsigned)u / (unsigned)cur.nu) : (int)(u / cur.nu);
    cur.u = (int)(u - (long long)pair * cur.nu);
    cur.kvh = pair / a.groups;
    cur.grp = pair - cur.kvh * a.groups;
  }
  Cursor ld = cur;
  int tiles = 2 * left;  // to be loaded
  int ids[kRuns];
#pragma unroll
  for (int i = 0; i < kRuns; ++i) ids[i] = -1;
  bool ld_v = false, withhold = g_gqa_test_stall != 0 && tid == 0;
  Pages pages = {-1, -1, -1, -1, 1.f, 1.f};
  Info<kUnit> now, next;  // of the unit at `cur`, and of the one behind it
  auto load_next = [&](int slot) {  // K of the unit at `ld`, the next time its V
    if (tiles == 0) return;
    --tiles;
    if (!ld_v) {
      fetch_pages<kUnit, true>(a, pages, ld.b, ld.kvh, ld.u, ld.len);
      next.held = 0;
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        const int from = (ld.u - pages.base) * kRuns + i;
        ids[i] = __shfl_sync(0xffffffffu, pages.id, from);
        next.held |= (ids[i] >= 0 ? 1 : 0) << i;
      }
      if (lane == 0 && !withhold) load_tile<D, kUnit>(a, &tk, ids, ld.kvh, ld.u, ring + slot * kTile, &full[slot]);
      withhold = false;
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {  // after the load: these may still be on their way
        const int from = (ld.u - pages.base) * kRuns + i;
        next.ks[i] = __shfl_sync(0xffffffffu, pages.ks, from);
        next.vs[i] = __shfl_sync(0xffffffffu, pages.vs, from);
      }
    } else {
      if (lane == 0) load_tile<D, kUnit>(a, &tv, ids, ld.kvh, ld.u, ring + slot * kTile, &full[slot]);
      advance(ld);
    }
    ld_v = !ld_v;
  };
  const int rows = a.g * a.s_q;
  RawQ<D> raw[NT];
  if (left > 0) {  // the first rows of q, ahead of the tiles that would be in their way
#pragma unroll
    for (int n = 0; n < NT; ++n) fetch_q<T, D>(a, cur.b, cur.kvh, cur.grp * kRows + 8 * n, rows, raw[n]);
  }
  load_next(0);
  now = next;
#pragma unroll
  for (int s = 1; s < kSlots; ++s) load_next(s);

  uint32_t q[NT][kSteps][2];
  float factor[NT][2];
  float o[kSteps][NT][4];  // (dim col(g) + 2 i, rows 2c, 2c + 1), (dim col(g) + 2 i + 1, the same), in units of sh.unit
  float m[NT][2], l[NT][2];
  int from = 0, q_first = 0, q_of[NT][2];  // the first row's query, and those of rows 2c, 2c + 1
  bool fresh = true, ok = true, first = true;
  if (left > 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n) scale_q<T, D>(a, raw[n], q[n], factor[n]);
  }
  bool q_ready = true;
  int slot = 0;
  uint32_t phase = 0;
  auto next_slot = [&]() {
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  };

  while (left > 0) {
    const int r0 = cur.grp * kRows;
    if (fresh) {
      if (!q_ready) {
#pragma unroll
        for (int n = 0; n < NT; ++n) load_q<T, D>(a, cur.b, cur.kvh, r0 + 8 * n, rows, q[n], factor[n]);
      }
      q_ready = false;
      q_first = r0 / a.g;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          m[n][k] = -INFINITY;
          l[n][k] = 0.f;
          q_of[n][k] = (r0 + 8 * n + 2 * c + k) / a.g;
        }
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
      sh.unit[warp] = sh.least_unit[warp] = 0.f;
      from = cur.u;
      fresh = false;
    }
    // positions below `all` are seen by every row, those from `len` on by none
    const int t0 = cur.u * kUnit;
    const int all = min(cur.len, cur.end + q_first);
    bool edge = t0 + kUnit > all || now.held != (1 << kRuns) - 1;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) edge |= now.vs[i] == 0.f;
    if (!(ok = mbar_wait_warp(&full[slot], phase, &sh.abort, &g_gqa_status))) break;

    // s^T: s[mt][n]: positions 16 mt + perm(g) (0, 1) and 8 further (2, 3), rows 2c, 2c + 1
    float s[kRuns][NT][4];
#pragma unroll
    for (int mt = 0; mt < kRuns; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[mt][n][0] = s[mt][n][1] = s[mt][n][2] = s[mt][n][3] = 0.f;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint32_t f[4][4];
        k_frags<D>(ring + slot * kTile, mt, h, f);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_f16(s[mt][n], f[k][0], f[k][1], f[k][2], f[k][3], q[n][4 * h + k][0], q[n][4 * h + k][1]);
      }
    }
    __syncwarp();
    load_next(slot);
    next_slot();

#pragma unroll
    for (int mt = 0; mt < kRuns; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float f = factor[n][k] * now.ks[mt];
          s[mt][n][k] *= f;
          s[mt][n][2 + k] *= f;
        }
    if (edge) {
#pragma unroll
      for (int mt = 0; mt < kRuns; ++mt) {
        const bool there = (now.held >> mt) & 1;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int lim = min(cur.len, cur.end + q_of[n][k]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!there || t0 + mt * 16 + h * 8 + Lay<D>::perm(g) >= lim) s[mt][n][2 * h + k] = -INFINITY;
          }
      }
    }
    // the rows' m, moved only where a score outgrows one by 2^15
    float top[NT][2];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        top[n][k] = fmaxf(s[0][n][k], s[0][n][2 + k]);
#pragma unroll
        for (int mt = 1; mt < kRuns; ++mt) top[n][k] = fmaxf(top[n][k], fmaxf(s[mt][n][k], s[mt][n][2 + k]));
        grew |= top[n][k] > m[n][k] + (kBelow + kRescale);
      }
    if (__any_sync(0xffffffffu, grew)) {
      float alpha[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float t = top[n][k];
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
          t -= kBelow;
          alpha[n][k] = 1.f;
          if (t > m[n][k]) {
            alpha[n][k] = fast_exp2(m[n][k] - t);
            m[n][k] = t;
            l[n][k] *= alpha[n][k];
          }
        }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][n][k] *= alpha[n][k & 1];
    }
    uint32_t p[kRuns][NT][2];  // p^T: rows g, positions 2c, 2c + 1 (of 8 and of the 8 further)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float base[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int mt = 0; mt < kRuns; ++mt) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[mt][n][k] = fast_exp2(s[mt][n][k] - base[k & 1]);
        l[n][0] += s[mt][n][0] + s[mt][n][2];
        l[n][1] += s[mt][n][1] + s[mt][n][3];
        p[mt][n][0] = transpose8(pack_half(s[mt][n][0], s[mt][n][1]));
        p[mt][n][1] = transpose8(pack_half(s[mt][n][2], s[mt][n][3]));
      }
    }
    if (!(ok = mbar_wait_warp(&full[slot], phase, &sh.abort, &g_gqa_status))) break;
    const uint32_t v_tile = ring + slot * kTile;
    float v_unit = sh.unit[warp];
#pragma unroll
    for (int mt = 0; mt < kRuns; ++mt) {
      // o into units of these positions' v_scale (0: they add nothing) unless it
      // is too small for one; a factor below 2^-126 would lose digits that o has
      const bool there = (now.held >> mt) & 1 && now.vs[mt] != 0.f;
      if (there && now.vs[mt] != v_unit) {  // the same in all lanes
        const float least = sh.least_unit[warp], size = fabsf(now.vs[mt]);
        if (size < least) {
          edge = true;
        } else {
          sh.least_unit[warp] = fmaxf(least, size * kUnitSpan);
#pragma unroll 1
          for (int i = 0; i < 3 && v_unit != now.vs[mt]; ++i) {
            const bool far = fabsf(v_unit) * 0x1p100f < size && v_unit != 0.f;
            const float next = far ? v_unit * 0x1p100f : now.vs[mt], r = far ? 0x1p-100f : v_unit / next;
            v_unit = next;
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][n][k] *= r;
          }
        }
      }
      // the four positions whose p this thread holds
      const int row[4] = {16 * mt + Lay<D>::perm(2 * c), 16 * mt + Lay<D>::perm(2 * c + 1),
                          16 * mt + 8 + Lay<D>::perm(2 * c), 16 * mt + 8 + Lay<D>::perm(2 * c + 1)};
      uint32_t w[4][D / 32];
#pragma unroll
      for (int k = 0; k < 4; ++k) lds_v_row<D>(v_tile, row[k], g, w[k]);
      // A position that some row does not see stays out of the product:
      // 0 * NaN of a stale or masked value would reach that row.  Zero
      // values here, added below for the rows that see them; so are those of
      // a scale below the unit.
      if (edge) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool in = there && now.vs[mt] == v_unit && t0 + row[k] < all;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) w[k][e] = in ? w[k][e] : 0u;
        }
      }
#pragma unroll
      for (int e = 0; e < D / 32; ++e) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t lo = __byte_perm(w[0][e], w[1][e], x ? 0x7362 : 0x5140);
          const uint32_t hi = __byte_perm(w[2][e], w[3][e], x ? 0x7362 : 0x5140);
          uint32_t a0, a1, a2, a3;
          widen4(lo, a0, a1);
          widen4(hi, a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[2 * e + x][n], a0, a1, a2, a3, p[mt][n][0], p[mt][n][1]);
        }
      }
      if (edge && there) {
        // the drafts' own positions (at most s_q - 1), or all of a scale below
        // the unit if they hold anything, one by one
        int lo = max(all, 0);
        if (now.vs[mt] != v_unit) {
          uint32_t any = 0;
#pragma unroll 1
          for (int x = c; x < 16; x += 4) {
            uint32_t v[D / 32];
            lds_v_row<D>(v_tile, 16 * mt + x, g, v);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) any |= v[e] & 0x7F7F7F7Fu;
          }
          if (__any_sync(0xffffffffu, any != 0)) lo = 0;
        }
        lo = max(lo, t0 + 16 * mt);
        const int hi = min(cur.len, t0 + 16 * mt + 16);
        const float by = now.vs[mt] / v_unit;
        for (int x = lo; x < hi; ++x) {
          const int in8 = (x - t0) & 7, h = ((x - t0) >> 3) & 1;
          const int from_lane = Lay<D>::unperm(in8) * 4 + c;
          uint32_t v[D / 32];
          lds_v_row<D>(v_tile, x - t0, g, v);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float px = by * __shfl_sync(0xffffffffu, h ? s[mt][n][2 + k] : s[mt][n][k], from_lane);
              if (x < cur.end + q_of[n][k]) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                  const uint32_t two = widen((v[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
                  const float2 val = __half22float2(*reinterpret_cast<const __half2*>(&two));
                  o[i][n][k] += px * val.x;
                  o[i][n][2 + k] += px * val.y;
                }
              }
            }
        }
      }
    }
    sh.unit[warp] = v_unit;
    __syncwarp();
    now = next;
    load_next(slot);
    next_slot();
    --left;
    const bool done = cur.u + 1 == cur.nu;  // the (sequence, head, group) ends here
    if (done || left == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 4);
          l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 8);
          l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 16);
        }
      const bool whole = from == 0 && done;
      const int piece = 2 * warp + (first ? 0 : 1);
      float* keep = left == 0 ? reinterpret_cast<float*>(smem + warp * kSlots * kTile) : first_o(warp);
      if (!whole && lane == 0) {
        sh.id[piece] = (cur.b * a.h_kv + cur.kvh) * a.groups + cur.grp;
        sh.from[piece] = from;
        sh.to[piece] = cur.u + 1;
        sh.nu[piece] = cur.nu;
        sh.in_ring[piece] = left == 0;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = 8 * n + 2 * c + k, r = r0 + row;
          const bool none = l[n][k] == 0.f;
          const float inv = none ? 0.f : 1.f / l[n][k];
          float v[2 * kSteps];
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {  // (v_unit / l might not be a normal number)
            v[2 * i] = o[i][n][k] * inv * v_unit;
            v[2 * i + 1] = o[i][n][2 + k] * inv * v_unit;
          }
          if (whole) {
            if (r < rows) {
              T* p = out_row<T>(a, cur.b, cur.kvh, r) + Lay<D>::col(g);
#pragma unroll
              for (int e = 0; e < 2 * kSteps; e += 8)
                *reinterpret_cast<uint4*>(p + e) = make_uint4(pack16<T>(v[e], v[e + 1]), pack16<T>(v[e + 2], v[e + 3]),
                                                              pack16<T>(v[e + 4], v[e + 5]), pack16<T>(v[e + 6], v[e + 7]));
              if (g == 0) *lse_at(a, cur.b, cur.kvh, r) = none ? -INFINITY : (m[n][k] + log2f(l[n][k])) * kLn2;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2 * kSteps; e += 4)
              *reinterpret_cast<float4*>(keep + row * D + Lay<D>::col(g) + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            if (g == 0) {
              sh.ml[piece][row] = m[n][k];
              sh.ml[piece][kRows + row] = l[n][k];
            }
          }
        }
      first = false;
      fresh = true;
    }
    advance(cur);
  }
  if (!ok) drain(full, kSlots, slot, phase, 2 * left - tiles);
  __syncthreads();

  // The CTA's pieces in order of the list (warp 0's first and last, warp 1's,
  // ...): sh.list_of; runs of one id are joined.
  static_assert(2 * kWarps <= 32, "one lane per piece");
  if (warp == 0) {
    const int id = lane < 2 * kWarps ? sh.id[lane] : -1;
    const unsigned there = __ballot_sync(0xffffffffu, id >= 0), before = there & ((1u << lane) - 1u);
    const int id_before = __shfl_sync(0xffffffffu, id, before ? 31 - __clz(before) : 0);
    const bool begins = id >= 0 && (!before || id_before != id);
    const unsigned runs = __ballot_sync(0xffffffffu, begins);
    if (id >= 0) sh.list_of[__popc(before)] = lane;
    if (begins) sh.run[__popc(runs & ((1u << lane) - 1u))] = __popc(before);
    if (lane == 0) {
      sh.n_runs = __popc(runs);
      sh.run[__popc(runs)] = __popc(there);
    }
  }
  Partial<D, NT>* mine = reinterpret_cast<Partial<D, NT>*>(a.ws) + (int64_t)blockIdx.x * 2;
  if (tid < 2) mine[tid].id = -1;
  __syncthreads();
  if (sh.abort) return;
  for (int x = tid; x < sh.n_runs * (kRows * D / 4); x += C::kThreads) {
    const int run = x / (kRows * D / 4), e = x % (kRows * D / 4) * 4;
    const int p0 = sh.run[run], n = sh.run[run + 1] - p0;
    const int head = sh.list_of[p0], last = sh.list_of[p0 + n - 1], id = sh.id[head];
    const bool begins = sh.from[head] == 0, ends = sh.to[last] == sh.nu[last];
    Partial<D, NT>* part = begins && ends ? nullptr : mine + (begins ? 1 : 0);
    join<T, D, NT>(a, e, n, id, [&](int i) -> const float* { return sh.ml[sh.list_of[p0 + i]]; },
                   [&](int i) -> const float* {
                     const int p = sh.list_of[p0 + i];
                     return sh.in_ring[p] ? reinterpret_cast<const float*>(smem + (p >> 1) * kSlots * kTile)
                                          : first_o(p >> 1);
                   },
                   part);
    if (part && e == 0) {
      part->id = id;
      part->last = 0;
      if (!ends) {
        const long long here = split.begin(first_part + (last >> 1) + 1);  // the list position behind it
        part->last = split.holder(here + (sh.nu[last] - sh.to[last]) - 1) / kWarps;
      }
    }
  }
}

// Joins what several CTAs have of one (sequence, head, group): CTA i's, if
// it begins there.  The pieces lie in the CTAs up to `last` (a short list
// leaves some of them without a unit).
constexpr int kJoinThreads = 256;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) gqa_join_kernel(const GqaArgs a) {
  constexpr int kRows = 8 * NT;
  __shared__ float ml[kMaxCtas][2 * kRows];
  __shared__ int there[kMaxCtas];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Partial<D, NT>* all = reinterpret_cast<const Partial<D, NT>*>(a.ws);
  const Partial<D, NT>* p = all + (int64_t)blockIdx.x * 2 + 1;
  const int id = p->id, n = p->last - (int)blockIdx.x + 1;
  if (id < 0) return;
  auto piece = [&](int i) { return i == 0 ? p : all + (int64_t)(blockIdx.x + i) * 2; };
  for (int k = threadIdx.x; k < n * kRows; k += kJoinThreads) {
    const int i = k / kRows, row = k % kRows;
    const Partial<D, NT>* x = piece(i);
    const bool is = x->id == id;
    const float xm = x->m[row], xl = x->l[row];
    ml[i][row] = is ? xm : -INFINITY;
    ml[i][kRows + row] = is ? xl : 0.f;
    if (row == 0) there[i] = is;
  }
  __syncthreads();
  for (int e = threadIdx.x * 4; e < kRows * D; e += kJoinThreads * 4)
    join<T, D, NT>(a, e, n, id, [&](int i) -> const float* { return ml[i]; },
                   // one that is not there has no values: any of this id do, its factor is 0
                   [&](int i) -> const float* { return there[i] ? piece(i)->o : p->o; }, (Partial<D, NT>*)nullptr);
}

// ------------------------------------------------------------------ weights
// lse of row r in log2 units; +inf, which makes its p 0, for a row that is
// not there or that saw nothing.
__device__ __forceinline__ float lse_log2(const GqaArgs& a, int b, int kvh, int r, int rows) {
  if (r >= rows) return INFINITY;
  const float x = __ldg(a.lse_in + ((int64_t)b * a.h_q + kvh * a.g + r % a.g) * a.s_q + r / a.g) * kLog2e;
  return x == -INFINITY ? INFINITY : x;
}

// Zeros behind every context, a warp for 512 positions at a time; this warp is the
// `me`-th of n.
__device__ __forceinline__ void zero_behind(const GqaArgs& a, int me, int n) {
  constexpr int kSpan = 512;
  const int lane = threadIdx.x & 31, spans = (a.width + kSpan - 1) / kSpan;
  const long long items = (long long)a.b * a.h_kv * spans;
  for (long long x = me; x < items; x += n) {
    const int row = items < (1ll << 31) ? (int)((unsigned)x / (unsigned)spans) : (int)(x / spans);
    const int from = (int)(x - (long long)row * spans) * kSpan, to = min(from + kSpan, a.width);
    const int len = held_len(a, row / a.h_kv);
    if (len >= to) continue;
    float* w = a.weights + (int64_t)(row / a.h_kv) * a.stride_w_b + (int64_t)(row % a.h_kv) * a.stride_w_h;
    if (len <= from && to - from == kSpan && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
#pragma unroll
      for (int t = 0; t < kSpan; t += 128) *reinterpret_cast<float4*>(w + from + t + 4 * lane) = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      for (int t = max(from, len) + lane; t < to; t += 32) w[t] = 0.f;
    }
  }
}

// A walk over a piece's (sequence, KV head) pairs.
template <int U>
struct Walk {
  int b, kvh, nu, len, end;  // nu: the pair's units; `end`: positions that its first query sees
  int from, n;               // the piece's units of this pair
  long long left;            // the piece's units from there on
  __device__ __forceinline__ void enter(const GqaArgs& a) {  // b, kvh, from and left are set
    len = held_len(a, b);
    end = __ldg(a.ctx + b) - a.s_q + 1;
    nu = units_of<U>(len);
    n = (int)min(left, (long long)(nu - from));
  }
  // The i-th piece of the list, of `pieces` places that were found; left == 0: it is empty.
  template <int W>
  __device__ __forceinline__ void begin(const GqaArgs& a, const ListShared<W>& list, int parts, int part, int i) {
    const Split split(list.total, parts);
    left = split.each + (part < split.more ? 1 : 0);
    if (left == 0) return;
    b = list.b[i];
    const int per_head = units_of<U>(held_len(a, b));
    const long long u = list.u[i];
    kvh = u < (1ll << 31) ? (int)((unsigned)u / (unsigned)per_head) : (int)(u / per_head);
    from = (int)(u - (long long)kvh * per_head);
    enter(a);
  }
  __device__ __forceinline__ bool next(const GqaArgs& a) {  // false: the piece ends
    left -= n;
    if (left == 0) return false;
    from = 0;
    if (++kvh == a.h_kv) {
      kvh = 0;
      ++b;
    }
    enter(a);
    return true;
  }
};

// Up to 8 rows (one n-tile of mma.sync): every warp of the grid takes a
// contiguous piece of the units of all (sequence, KV head) pairs and keeps the
// rows' q in registers.  A thread adds p of its rows, then the four c are
// joined by a halving exchange that leaves one position per lane.  Bound by
// its start and K's bytes: 32 sequences of 500 to 16,384, 8 KV heads, d = 64
// (95 MB) 30 us.
template <int D>
struct Wts {
  static constexpr int kUnit = 64;
  static constexpr int kWarps = 12;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = kUnit * D;
  static constexpr int kSlots = 2;
};
template <int D>
struct WeightsShared {
  uint64_t full[Wts<D>::kWarps][Wts<D>::kSlots];
  ListShared<Wts<D>::kWarps> list;
  int abort;
};
template <int D>
constexpr int weights_smem() {
  using C = Wts<D>;
  return 1024 + C::kWarps * C::kSlots * C::kTile + (int)sizeof(WeightsShared<D>);
}

template <typename T, int D>
__global__ void __launch_bounds__(Wts<D>::kThreads, 1)
gqa_weights_kernel(const __grid_constant__ CUtensorMap tk, const GqaArgs a) {
  using C = Wts<D>;
  constexpr int kWarps = C::kWarps, kSlots = C::kSlots, kTile = C::kTile, kSteps = D / 16;
  constexpr int kUnit = C::kUnit, kRuns = kUnit / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  WeightsShared<D>& sh = *reinterpret_cast<WeightsShared<D>*>(smem + kWarps * kSlots * kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem + warp * kSlots * kTile);
  uint64_t* full = sh.full[warp];
  if (lane == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(&full[s], 1);
    fence_mbarrier_init();
  }
  if (tid == 0) sh.abort = 0;
  const int rows = a.g * a.s_q;
  const int parts = gridDim.x * kWarps;
  find_places<kWarps, kUnit>(a, a.h_kv, blockIdx.x * kWarps, kWarps, parts, sh.list);
  Walk<kUnit> cur = {};
  cur.begin(a, sh.list, parts, blockIdx.x * kWarps + warp, warp);

  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  uint32_t q[kSteps][2];
  float factor[2], lse2[2];
  Info<kUnit> now, next;  // of the unit at the products' cursor, and of the one behind it
  Walk<kUnit> ld = cur;
  int ld_u = 0;  // of ld.n
  bool more = cur.left > 0;
  int loaded = 0;  // and not yet used
  Pages pages = {-1, -1, -1, -1, 1.f, 1.f};
  auto load_next = [&](int to) {
    if (more && ld_u == ld.n) {
      more = ld.next(a);
      ld_u = 0;
    }
    if (!more) return;
    const int u = ld.from + ld_u;
    fetch_pages<kUnit, false>(a, pages, ld.b, ld.kvh, u, ld.len);
    int ids[kRuns];
    next.held = 0;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      ids[i] = __shfl_sync(0xffffffffu, pages.id, (u - pages.base) * kRuns + i);
      next.held |= (ids[i] >= 0 ? 1 : 0) << i;
    }
    if (lane == 0) load_tile<D, kUnit>(a, &tk, ids, ld.kvh, u, ring + to * kTile, &full[to]);
#pragma unroll
    for (int i = 0; i < kRuns; ++i)  // after the load: these may still be on their way
      next.ks[i] = __shfl_sync(0xffffffffu, pages.ks, (u - pages.base) * kRuns + i);
    ++ld_u;
    ++loaded;
  };
  RawQ<D> raw;  // the first rows of q, ahead of the tiles that would be in their way
  if (more) fetch_q<T, D>(a, cur.b, cur.kvh, 0, rows, raw);
  load_next(slot);
  now = next;
  load_next((slot + 1) % kSlots);
  if (!a.accumulate) zero_behind(a, blockIdx.x * kWarps + warp, gridDim.x * kWarps);  // while the first tiles come
  bool go = cur.left > 0, q_ready = true;
  if (go) scale_q<T, D>(a, raw, q, factor);
  while (go && ok) {  // the pairs of the piece, one after another
    if (!q_ready) load_q<T, D>(a, cur.b, cur.kvh, 0, rows, q, factor);
    q_ready = false;
    lse2[0] = lse_log2(a, cur.b, cur.kvh, 2 * c, rows);
    lse2[1] = lse_log2(a, cur.b, cur.kvh, 2 * c + 1, rows);
    // a row that saw nothing adds nothing, whatever its scores are
    const bool left_out = __any_sync(0xffffffffu, (2 * c < rows && lse2[0] == INFINITY) ||
                                                      (2 * c + 1 < rows && lse2[1] == INFINITY));
    for (int j = 0; j < cur.n; ++j) {
      const int t0 = (cur.from + j) * kUnit;
      const bool edge = left_out || t0 + kUnit > min(cur.len, cur.end) || now.held != (1 << kRuns) - 1;
      // the positions whose weights this lane will hold
      const int t_mine = t0 + 8 * c + Lay<D>::perm(g);
      float* w = a.weights + (int64_t)cur.b * a.stride_w_b + (int64_t)cur.kvh * a.stride_w_h + t_mine;
      float before[kUnit / 32];
#pragma unroll
      for (int x = 0; x < kUnit / 32; ++x) {
        const int t = t_mine + 32 * x;
        before[x] = a.accumulate && t < cur.len && t < a.width ? w[32 * x] : 0.f;
      }
      if (!(ok = mbar_wait_warp(&full[slot], phase, &sh.abort, &g_gqa_status))) break;
      uint32_t f[4][4];
      float s[kRuns][4];
#pragma unroll
      for (int mt = 0; mt < kRuns; ++mt) {
        s[mt][0] = s[mt][1] = s[mt][2] = s[mt][3] = 0.f;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          k_frags<D>(ring + slot * kTile, mt, h, f);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16(s[mt], f[k][0], f[k][1], f[k][2], f[k][3], q[4 * h + k][0], q[4 * h + k][1]);
        }
      }
      __syncwarp();
      --loaded;
      const Info<kUnit> here = now;
      now = next;
      load_next(slot);
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
      float sum[2 * kRuns];  // positions 8 i + perm(g)
      if (!edge) {
#pragma unroll
        for (int i = 0; i < 2 * kRuns; ++i)
          sum[i] = fast_exp2(fmaf(s[i >> 1][2 * (i & 1)], factor[0] * here.ks[i >> 1], -lse2[0])) +
                   fast_exp2(fmaf(s[i >> 1][2 * (i & 1) + 1], factor[1] * here.ks[i >> 1], -lse2[1]));
      } else {
#pragma unroll
        for (int i = 0; i < 2 * kRuns; ++i) sum[i] = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int lim = lse2[k] == INFINITY ? INT_MIN : cur.end + (2 * c + k) / a.g;
#pragma unroll
          for (int i = 0; i < 2 * kRuns; ++i) {
            const bool there = (here.held >> (i >> 1)) & 1;
            const float p = fast_exp2(fmaf(s[i >> 1][2 * (i & 1) + k], factor[k] * here.ks[i >> 1], -lse2[k]));
            sum[i] += there && t0 + 8 * i + Lay<D>::perm(g) < lim ? p : 0.f;
          }
        }
      }
      // four values over the four c: each step sends half of them
#pragma unroll
      for (int x = 0; x < kUnit / 32; ++x) {
#pragma unroll
        for (int h = 2; h >= 1; h >>= 1) {
          const bool up = lane & h;
#pragma unroll
          for (int i = 4 * x; i < 4 * x + h; ++i) {
            const float send = up ? sum[i] : sum[i + h], keep = up ? sum[i + h] : sum[i];
            sum[i] = keep + __shfl_xor_sync(0xffffffffu, send, h);
          }
        }
        const int t = t_mine + 32 * x;
        if (t < cur.len && t < a.width) w[32 * x] = before[x] + sum[4 * x];
      }
    }
    go = cur.next(a);
  }
  if (!ok) drain(full, kSlots, slot, phase, loaded);
}

// More rows: S = K q^T on tcgen05, 128 positions by up to 128 rows (further
// rows take further passes).  A TMEM lane is a position, so a thread has all
// rows' scores of one and adds their p by itself, without an exchange; K
// becomes fp16 on its way from shared memory to TMEM (the A operand), a row of
// a tile per thread, and q stands in shared memory, scaled as above.  A CTA
// takes a contiguous piece of the list:
//   warps 0-11      p of every third unit a group of four, and their sums;
//   warps 12-15     q's rows, and K's conversion;
//   warp 16         page ids, scales, K's loads;     warp 17  the MMAs.
// TMEM: K of two units (2 x 64 columns), S of three (3 x 128).
//
// With many rows the exponentials bound it, 16 a cycle and SM: 128 rows of
// 105,000 positions and 8 heads are 108 M of them, 27 us; it takes 60, of
// which 6 pass before the first S.  (S in tiles of 64 rows took 63: an MMA
// whose A is in TMEM takes 64 cycles whatever N is.  Two groups: 68.)  With
// few it is K's bytes.  mma.sync, an n-tile of rows after another, was the
// quicker only up to 16 rows.  32 sequences of 16,000, d = 128, us (this;
// mma.sync):  8 rows 115, 104;  16 117, 114;  32 122, 152;  128 199, 397.
constexpr int kWinUnit = 128, kWinRows = 128;
constexpr int kWinStages = 8;  // K tiles
// Groups and S buffers: as many, so that a group that waits for its next unit
// has seen the buffer's last one complete (a parity tells only two apart).
constexpr int kWinGroups = 3;
constexpr int kWinInfos = 16;  // more than units can lie between load and sums: 8 + 2 + 3
constexpr int kWinConvert = 4 * kWinGroups, kWinLoad = kWinConvert + 4, kWinMma = kWinLoad + 1, kWinWarps = kWinMma + 1;
struct WindowShared {
  float factor[2][kWinRows], minus_lse[2][kWinRows];
  float common[2][kWinRows / 32];  // the factor of 32 rows; 0: each has its own, or some are left out
  uint64_t k_full[kWinStages], k_empty[kWinStages], a_full[2], a_empty[2], s_full[kWinGroups], s_empty[kWinGroups];
  uint64_t q_full[2], q_empty[2], done;
  ListShared<kWinWarps> list;
  Walk<kWinUnit> first;
  float ks[kWinInfos][kWinUnit / 16];
  int held[kWinInfos];
  uint32_t tmem;
  int abort;
};
template <int D>
constexpr int window_smem() {
  return 1024 + 2 * kWinRows * D * 2 + kWinStages * kWinUnit * D + (int)sizeof(WindowShared);
}

template <typename T, int D>
__global__ void __launch_bounds__(kWinWarps * 32, 1)
gqa_window_weights_kernel(const __grid_constant__ CUtensorMap tk, const GqaArgs a) {
  constexpr int kTile = kWinUnit * D, kQ = kWinRows * D * 2, kQChunk = kWinRows * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  WindowShared& sh = *reinterpret_cast<WindowShared*>(smem + 2 * kQ + kWinStages * kTile);
  const uint32_t q_s = smem_u32(smem), ring = q_s + 2 * kQ;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kWinStages; ++i) {
      mbar_init(&sh.k_full[i], 2);
      mbar_init(&sh.k_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.a_full[i], 4);
      mbar_init(&sh.a_empty[i], 1);
      mbar_init(&sh.q_full[i], 4);
      mbar_init(&sh.q_empty[i], 1 + kWinConvert);
    }
    for (int i = 0; i < kWinGroups; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_empty[i], 4);
    }
    mbar_init(&sh.done, 1);
    sh.abort = 0;
    fence_mbarrier_init();
  }
  if (warp == kWinMma) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  find_places<kWinWarps, kWinUnit>(a, a.h_kv, blockIdx.x, 1, gridDim.x, sh.list);  // synchronises
  tc_fence_after();
  const uint32_t tmem = sh.tmem, tmem_s = tmem + 128;
  if (tid == 0) sh.first.begin(a, sh.list, gridDim.x, blockIdx.x, 0);
  __syncthreads();
  const int rows = sh.first.left > 0 ? a.g * a.s_q : 0;  // an empty piece has nothing to do
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_warp(bar, parity, &sh.abort, &g_gqa_status); };
  auto arrive = [&](uint64_t* bar) {  // the warp's
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  bool ok = true;
  int nu = 0, np = 0;  // units and pairs so far

  if (warp < kWinConvert) {
    // ------------------------------------------------------------------ p
    const int group = warp >> 2, p = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    if (!a.accumulate) zero_behind(a, blockIdx.x * kWinConvert + warp, gridDim.x * kWinConvert);
    for (int r0 = 0; r0 < rows && ok; r0 += kWinRows) {
      const int cols = (min(rows - r0, kWinRows) + 31) & ~31;
      const bool add = a.accumulate || r0 > 0;
      Walk<kWinUnit> x = sh.first;
      do {
        if (!(ok = wait(&sh.q_full[np & 1], (np >> 1) & 1))) break;
        const float* factor = sh.factor[np & 1];
        const float* minus_lse = sh.minus_lse[np & 1];
        for (int j = 0; j < x.n; ++j, ++nu) {
          const int buf = nu % kWinGroups;
          if (buf != group) continue;
          const int t = (x.from + j) * kWinUnit + p;
          float* w = a.weights + (int64_t)x.b * a.stride_w_b + (int64_t)x.kvh * a.stride_w_h + t;
          const bool live = t < x.len && t < a.width;
          uint64_t sum[2] = {0, 0};  // pairs of zeros
          if (!(ok = wait(&sh.s_full[buf], (nu / kWinGroups) & 1))) break;
          tc_fence_after();
          const int held = sh.held[nu % kWinInfos];
          const float ks = sh.ks[nu % kWinInfos][p >> 4];
          const bool edge = (x.from + j + 1) * kWinUnit > min(x.len, x.end + r0 / a.g) || held != 0xff;
          // rows before it do not see the position
          const int r_min = (held >> (p >> 4)) & 1 ? min(max(t - x.end + 1, 0), a.s_q) * a.g - r0 : INT_MAX;
          // 16 bytes of shared memory for every four scores (32 with each
          // row's own factor) are half of what the exponentials take
          auto add_up = [&](const float (&s)[32], int col, float by, auto general) {
            const uint64_t scale = pair(by, by);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 l = *reinterpret_cast<const float4*>(minus_lse + col + e);
              uint64_t t[2] = {pair(s[e], s[e + 1]), pair(s[e + 2], s[e + 3])}, by2[2] = {scale, scale};
              if constexpr (general) {
                const float4 f = *reinterpret_cast<const float4*>(factor + col + e);
                by2[0] = mul2(scale, pair(f.x, f.y));
                by2[1] = mul2(scale, pair(f.z, f.w));
              }
              float2 y[2] = {unpair(fma2(t[0], by2[0], pair(l.x, l.y))), unpair(fma2(t[1], by2[1], pair(l.z, l.w)))};
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                y[i].x = fast_exp2(y[i].x);
                y[i].y = fast_exp2(y[i].y);
                if constexpr (general) {
                  const float2 from = i ? make_float2(l.z, l.w) : make_float2(l.x, l.y);
                  y[i].x = col + e + 2 * i >= r_min && from.x != -INFINITY ? y[i].x : 0.f;
                  y[i].y = col + e + 2 * i + 1 >= r_min && from.y != -INFINITY ? y[i].y : 0.f;
                }
                sum[i] = add2(sum[i], pair(y[i].x, y[i].y));
              }
            }
          };
          for (int col = 0; col < cols; col += 32) {
            float s[32];
            tmem_ld32(tmem_s + lanes + buf * kWinRows + col, s);
            const float f = sh.common[np & 1][col / 32];
            tc_wait_ld();
            if (col + 32 >= cols) {
              tc_fence_before();
              arrive(&sh.s_empty[buf]);
            }
            if (edge || f == 0.f)
              add_up(s, col, ks, std::true_type());
            else
              add_up(s, col, ks * f, std::false_type());
          }
          const float2 v = unpair(add2(sum[0], sum[1]));
          if (live) *w = (add ? *w : 0.f) + (v.x + v.y);
        }
        if (!ok) break;
        arrive(&sh.q_empty[np & 1]);
        ++np;
      } while (x.next(a));
      // the next pass adds to what another group may have written (once per
      // pass by every warp, whether its waits gave up or not)
      if (r0 + kWinRows < rows) ok = !named_bar_or(1, kWinConvert * 32, !ok);
    }
  } else if (warp < kWinLoad) {
    // -------------------------------------------------------- q, conversion
    const int w4 = warp - kWinConvert;
    constexpr int kLanes = D / 8, kRowsOnce = 32 / kLanes;  // lanes of a row of q, rows of a load
    for (int r0 = 0; r0 < rows && ok; r0 += kWinRows) {
      const int cols = (min(rows - r0, kWinRows) + 31) & ~31;
      Walk<kWinUnit> x = sh.first;
      do {
        const int qb = np & 1;
        if (np >= 2 && !(ok = wait(&sh.q_empty[qb], ((np >> 1) - 1) & 1))) break;
        // 32 rows at a time, in two short passes (unrolled as one, its cold code
        // took longer than its loads): the 16-bit values as they are to where
        // they belong, then each thread's own in place.  Where the rows'
        // largest values are within 2^8 of one another they get one power of two.
        const int piece = lane % kLanes;
        for (int r1 = w4 * 32; r1 < cols; r1 += 4 * 32) {
          const T* q = static_cast<const T*>(a.q) + (int64_t)x.b * a.stride_q_b + (int64_t)x.kvh * a.g * a.stride_q_h + piece * 8;
          const int sub = lane / kLanes;
          const uint32_t to = q_s + qb * kQ + (piece >> 3) * kQChunk + (r1 + sub) * 128;  // + 128 a row
          auto at = [&](int i) { return to + i * kRowsOnce * 128 + (((piece & 7) ^ ((sub + i * kRowsOnce) & 7)) << 4); };
          auto row_top = [&](const uint4& w) {
            uint32_t top = largest<T>(w);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            return top;
          };
          int r = r0 + r1 + sub, row_q = r / a.g, row_h = r - row_q * a.g;
          uint32_t most = 0, least = 0xFFFFFFFFu;
          constexpr int kDeep = 4;
#pragma unroll 1
          for (int i = 0; i < kLanes; i += kDeep) {
            uint4 raw[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
              raw[k] = make_uint4(0, 0, 0, 0);
              if (r < rows) raw[k] = __ldg(reinterpret_cast<const uint4*>(q + (int64_t)row_q * a.stride_q_s + (int64_t)row_h * a.stride_q_h));
              r += kRowsOnce;
              row_h += kRowsOnce;
              while (row_h >= a.g) {
                row_h -= a.g;
                ++row_q;
              }
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
              sts_v4(at(i + k), raw[k]);
              const uint32_t top = row_top(raw[k]);
              most = max(most, top);
              least = min(least, top ? top : 0xFFFFFFFFu);
            }
          }
          const float minus_lse = -lse_log2(a, x.b, x.kvh, r0 + r1 + lane, rows);
          sh.minus_lse[qb][r1 + lane] = minus_lse;
          // a row that saw nothing adds nothing, whatever its scores are
          const bool left_out = __any_sync(0xffffffffu, r0 + r1 + lane < rows && minus_lse == -INFINITY);
          most = __reduce_max_sync(0xffffffffu, most);
          least = min(__reduce_min_sync(0xffffffffu, least), most);
          const bool one = !left_out && most < 0x7F800000u && __uint_as_float(least) * 256.f >= __uint_as_float(most);
          float up, down;
          row_scale(a, __uint_as_float(most), up, down);
#pragma unroll 2
          for (int i = 0; i < kLanes; ++i) {
            const uint4 w = lds_v4(at(i));
            if (!one) row_scale(a, __uint_as_float(row_top(w)), up, down);
            const float4 u = four<T>(make_uint2(w.x, w.y)), v = four<T>(make_uint2(w.z, w.w));
            sts_v4(at(i), make_uint4(pack_half(u.x * up, u.y * up), pack_half(u.z * up, u.w * up),
                                     pack_half(v.x * up, v.y * up), pack_half(v.z * up, v.w * up)));
            if (piece == 0) sh.factor[qb][r1 + sub + i * kRowsOnce] = down;
          }
          if (lane == 0) sh.common[qb][r1 / 32] = one ? down : 0.f;
        }
        fence_proxy_async_smem();
        arrive(&sh.q_full[qb]);
        ++np;
        for (int j = 0; j < x.n; ++j, ++nu) {
          const int st = nu % kWinStages, row = w4 * 32 + lane;
          if (!(ok = wait(&sh.k_full[st], (nu / kWinStages) & 1))) break;
          if (nu >= 2 && !(ok = wait(&sh.a_empty[nu & 1], ((nu >> 1) - 1) & 1))) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            uint4 k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = lds_v4(ring + st * kTile + Lay<D>::piece(row, 4 * i + e));
            float h[32];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t words[4] = {k[e].x, k[e].y, k[e].z, k[e].w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                uint32_t lo, hi;
                widen4(words[y], lo, hi);
                h[8 * e + 2 * y] = __uint_as_float(lo);
                h[8 * e + 2 * y + 1] = __uint_as_float(hi);
              }
            }
            tmem_st32(tmem + ((uint32_t)(w4 * 32) << 16) + (nu & 1) * 64 + i * 32, h);
          }
          arrive(&sh.k_empty[st]);
          tc_wait_st();
          tc_fence_before();
          arrive(&sh.a_full[nu & 1]);
        }
      } while (ok && x.next(a));
    }
  } else if (warp == kWinLoad) {
    // -------------------------------------------------------------- loads
    // 512 positions at a time, a lane for 16 of them: four units, whose blocks
    // are loaded by as many lanes at once (one lane for all took 1,300 cycles
    // of a unit).
    constexpr int kRuns = kWinUnit / 16, kUnits = 32 / kRuns;
    const int unit = lane / kRuns, run = lane % kRuns, box = min(a.page, kWinUnit);
    // every lane's stage is free (a unit's own one; the first ones are)
    auto wait_free = [&](int nth, int st) {
      const uint32_t bar = smem_u32(&sh.k_empty[st]), parity = (nth / kWinStages - 1) & 1;
      volatile int* abort = &sh.abort;
      const long long t0 = clock64();
      for (;;) {
        if (__all_sync(0xffffffffu, nth < kWinStages || mbar_try_wait(bar, parity))) return true;
        const bool late = clock64() - t0 > kWaitLimitCycles;
        if (__any_sync(0xffffffffu, late || *abort)) {
          *abort = 1;
          if (late) atomicOr(&g_gqa_status, kErrWaitTimeout);
          return false;
        }
      }
    };
    for (int r0 = 0; r0 < rows && ok; r0 += kWinRows) {
      Walk<kWinUnit> x = sh.first;
      do {
        for (int u0 = x.from & ~(kUnits - 1); u0 < x.from + x.n; u0 += kUnits) {
          const int u = u0 + unit, t = u * kWinUnit + run * 16;
          int id = -1;
          float ks = 1.f;
          if (t < x.len) {
            id = __ldg(a.table + (int64_t)x.b * a.stride_table + (t >> a.page_shift));
            if (id < 0 || id >= a.num_blocks) id = -1;
            if (id >= 0) ks = __ldg(a.k_scale + (int64_t)id * a.h_kv + x.kvh);
          }
          const int skip = max(x.from - u0, 0), n = min(x.from + x.n - u0, kUnits) - skip;
          const bool mine = unit >= skip && unit < skip + n;
          const int nth = nu + (mine ? unit - skip : 0), st = nth % kWinStages, slot = nth % kWinInfos;
          const unsigned held = __ballot_sync(0xffffffffu, id >= 0) >> (unit * kRuns) & 0xffu;
          const bool load = mine && id >= 0 && (run * 16 & (box - 1)) == 0;
          const unsigned loads = __ballot_sync(0xffffffffu, load) >> (unit * kRuns) & 0xffu;
          if (!(ok = wait_free(nth, st))) break;
          if (mine && run == 0) mbar_arrive_expect_tx(&sh.k_full[st], __popc(loads) * box * D);
          __syncwarp();
          if (load) tma_load_4d(ring + st * kTile + run * 16 * D, &tk, 0, t & (a.page - 1), x.kvh, id, &sh.k_full[st]);
          if (mine) sh.ks[slot][run] = ks;
          if (mine && run == 0) sh.held[slot] = (int)held;
          __syncwarp();
          if (mine && run == 0) mbar_arrive(&sh.k_full[st]);
          nu += n;
        }
      } while (ok && x.next(a));
    }
    if (sh.abort) {  // what is in flight lands (or its wait runs out) before the CTA's shared memory goes
      for (int x = max(0, nu - kWinStages); x < nu; ++x) {
        const long long t = clock64();
        while (!mbar_try_wait(smem_u32(&sh.k_full[x % kWinStages]), (x / kWinStages) & 1, 1000u) &&
               clock64() - t < kWaitLimitCycles) {
        }
      }
    }
  } else {
    // --------------------------------------------------------------- MMAs
    for (int r0 = 0; r0 < rows && ok; r0 += kWinRows) {
      const uint32_t idesc = idesc_of<__half>((min(rows - r0, kWinRows) + 31) & ~31, false);
      Walk<kWinUnit> x = sh.first;
      do {
        const int qb = np & 1;
        if (!(ok = wait(&sh.q_full[qb], (np >> 1) & 1))) break;
        for (int j = 0; j < x.n; ++j, ++nu) {
          const int buf = nu % kWinGroups;
          if (nu >= kWinGroups && !(ok = wait(&sh.s_empty[buf], (nu / kWinGroups - 1) & 1))) break;
          if (!(ok = wait(&sh.a_full[nu & 1], (nu >> 1) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t b = desc_low(q_s + qb * kQ, 16);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_ts(tmem_s + buf * kWinRows, tmem + (nu & 1) * 64 + kk * 8, b + (kk >> 2) * (kQChunk >> 4) + (kk & 3) * 2,
                      kSw128High, idesc, kk != 0);
            umma_commit(&sh.s_full[buf]);
            umma_commit(&sh.a_empty[nu & 1]);
            if (j + 1 == x.n) umma_commit(&sh.q_empty[qb]);
          }
          __syncwarp();
        }
        ++np;
      } while (ok && x.next(a));
    }
    // every MMA has completed before TMEM is freed
    if (elect_one()) umma_commit(&sh.done);
    __syncwarp();
    const long long t = clock64();
    while (!mbar_try_wait(smem_u32(&sh.done), 0, 1000u) && clock64() - t < kWaitLimitCycles) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWinMma) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ host
// [num_blocks][h_kv][page][d] of one byte, boxes of up to `unit` rows of a head.
bool make_map(CUtensorMap* m, const void* base, int64_t stride_block, int64_t stride_row, int64_t stride_head,
              int unit, const dsv4b_gqa_cache& c) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c.d, (cuuint64_t)c.page_block_size, (cuuint64_t)c.h_kv,
                              (cuuint64_t)c.num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)stride_row, (cuuint64_t)stride_head, (cuuint64_t)stride_block};
  const cuuint32_t box[4] = {(cuuint32_t)c.d, (cuuint32_t)(c.page_block_size < unit ? c.page_block_size : unit), 1, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, c.d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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

template <typename T, int D, int NT>
cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, GqaArgs a, int grid, cudaStream_t stream) {
  using C = Dec<D, NT>;
  constexpr int smem = decode_smem<D, NT>();
  static_assert(smem <= 227 * 1024, "decode kernel shared memory");
  static bool done[64] = {};
  cudaError_t e = allow_smem(&gqa_decode_kernel<T, D, NT>, smem, done);
  if (e != cudaSuccess) return e;
  a.groups = (a.g * a.s_q + C::kRows - 1) / C::kRows;
  gqa_decode_kernel<T, D, NT><<<grid, C::kThreads, smem, stream>>>(tk, tv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;  // its launch overlaps the decode; it waits in the kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, gqa_join_kernel<T, D, NT>, a);
}

template <typename T, int D>
cudaError_t pick_decode(const CUtensorMap& tk, const CUtensorMap& tv, const GqaArgs& a, int grid, cudaStream_t stream) {
  return a.g * a.s_q <= 8 ? launch_decode<T, D, 1>(tk, tv, a, grid, stream)
                          : launch_decode<T, D, 2>(tk, tv, a, grid, stream);
}

template <typename T, int D>
cudaError_t launch_weights(const CUtensorMap& tk, const GqaArgs& a, int grid, cudaStream_t stream) {
  static_assert(weights_smem<D>() <= 227 * 1024 && window_smem<D>() <= 227 * 1024, "weights kernels' shared memory");
  static bool few_done[64] = {}, many_done[64] = {};
  cudaError_t e;
  if (a.g * a.s_q <= 8) {  // (one n-tile)
    if ((e = allow_smem(&gqa_weights_kernel<T, D>, weights_smem<D>(), few_done)) != cudaSuccess) return e;
    gqa_weights_kernel<T, D><<<grid, Wts<D>::kThreads, weights_smem<D>(), stream>>>(tk, a);
  } else {
    if ((e = allow_smem(&gqa_window_weights_kernel<T, D>, window_smem<D>(), many_done)) != cudaSuccess) return e;
    gqa_window_weights_kernel<T, D><<<grid, kWinWarps * 32, window_smem<D>(), stream>>>(tk, a);
  }
  return cudaGetLastError();
}

}  // namespace

size_t gqa_decode_ws_bytes(int sms, int d) {
  const int n = grid_of(sms);
  const size_t one = d == 128 ? ws_bytes<128, 1>(n) : ws_bytes<64, 1>(n);
  const size_t two = d == 128 ? ws_bytes<128, 2>(n) : ws_bytes<64, 2>(n);
  return one > two ? one : two;
}

cudaError_t launch_gqa_decode(const dsv4b_gqa_cache& c, const dsv4b_gqa_query& q, void* out, int64_t stride_o_b,
                              int64_t stride_o_s, int64_t stride_o_h, float* lse, void* ws, int sms,
                              cudaStream_t stream, int* bad_arg) {
  CUtensorMap tk, tv;
  constexpr int kUnit = Dec<128, 1>::kUnit;  // every variant's
  if (!make_map(&tk, c.k, c.stride_k_block, c.stride_k_row, c.stride_k_head, kUnit, c) ||
      !make_map(&tv, c.v, c.stride_v_block, c.stride_v_row, c.stride_v_head, kUnit, c)) {
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
    return c.d == 128 ? pick_decode<__nv_bfloat16, 128>(tk, tv, a, grid, stream)
                      : pick_decode<__nv_bfloat16, 64>(tk, tv, a, grid, stream);
  return c.d == 128 ? pick_decode<__half, 128>(tk, tv, a, grid, stream)
                    : pick_decode<__half, 64>(tk, tv, a, grid, stream);
}

cudaError_t launch_gqa_weights(const dsv4b_gqa_cache& c, const dsv4b_gqa_query& q, const float* lse, float* weights,
                               int64_t stride_w_b, int64_t stride_w_h, int width, int accumulate, int sms,
                               cudaStream_t stream, int* bad_arg) {
  GqaArgs a = make_args(c, q);
  CUtensorMap tk;
  const int unit = a.g * a.s_q <= 8 ? Wts<128>::kUnit : kWinUnit;
  if (!make_map(&tk, c.k, c.stride_k_block, c.stride_k_row, c.stride_k_head, unit, c)) {
    *bad_arg = 1;
    return cudaErrorInvalidValue;
  }
  a.lse_in = lse;
  a.weights = weights;
  a.stride_w_b = stride_w_b;
  a.stride_w_h = stride_w_h;
  a.width = width;
  a.accumulate = accumulate;
  const int grid = grid_of(sms);
  if (q.dtype == DSV4B_BF16)
    return c.d == 128 ? launch_weights<__nv_bfloat16, 128>(tk, a, grid, stream)
                      : launch_weights<__nv_bfloat16, 64>(tk, a, grid, stream);
  return c.d == 128 ? launch_weights<__half, 128>(tk, a, grid, stream) : launch_weights<__half, 64>(tk, a, grid, stream);
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
