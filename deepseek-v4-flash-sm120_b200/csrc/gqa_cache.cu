// The 8-bit grouped-query cache: append and eviction (include/dsv4b.h,
// dsv4b_gqa_cache_append and dsv4b_gqa_cache_evict).
//
// A block of page_block_size positions and a head share one scale s, so a
// value x is stored as e4m3(x / s).  The append rule takes s = 2^e, the
// smallest with amax <= 448 s: dividing by it is exact, so a stored value is
// rounded once, and when a later token raises e, moving the block's older
// rows to it only drops an exponent (exact but where they turn subnormal).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dsv4b.h"
#include "dsv4b_kernels.h"

namespace dsv4b {
namespace {

// ------------------------------------------------------------------ values
template <typename T>
__device__ __forceinline__ float2 to_f32x2(uint32_t w);
template <>
__device__ __forceinline__ float2 to_f32x2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 to_f32x2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The smallest e >= -100 with amax <= 448 * 2^e (448 = 1.75 * 2^8), read
// off the bits: amax = 1.m * 2^x, e = x - 8, one more if 1.m > 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int x = (int)(bits >> 23) - 127;
  return max(-100, x - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0));
}

__device__ __forceinline__ bool is_power_of_two(float s) {
  const uint32_t bits = __float_as_uint(s);
  const uint32_t x = bits >> 23;  // sign and exponent
  return (bits & 0x7FFFFFu) == 0 && x >= 1 && x <= 253;  // 1 / s is normal too
}

// Two fp32 to two e4m3 bytes (low byte first): nearest even, +-448 beyond.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// The larger of two 16-bit integers, in both halves.
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.s16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Two fp32 times r, at once (each an ordinary product).
__device__ __forceinline__ float2 scaled(float2 f, float r) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(f.x), "+f"(f.y)
      : "f"(r));
  return f;
}
// Sixteen e4m3 times r <= 1, rounded again.  A power of two from 2^-15 on
// keeps e4m3's values (multiples of 2^-9 up to 448) exact in fp16, so the
// product is rounded once there too; other factors go through fp32.
__device__ __forceinline__ uint32_t rescale_word_half(uint32_t w, __half2 r) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const __half2 a = __hmul2(*reinterpret_cast<__half2*>(&lo), r), b = __hmul2(*reinterpret_cast<__half2*>(&hi), r);
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f16x2 l, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 h, %2;\n\tmov.b32 %0, {l, h};\n\t}"
      : "=r"(d)
      : "r"(*reinterpret_cast<const uint32_t*>(&a)), "r"(*reinterpret_cast<const uint32_t*>(&b)));
  return d;
}
__device__ __forceinline__ uint32_t rescale_word(uint32_t w, float r) {
  const float2 a = scaled(from_e4m3x2(w & 0xFFFFu), r), b = scaled(from_e4m3x2(w >> 16), r);
  return to_e4m3x2(a.x, a.y) | (to_e4m3x2(b.x, b.y) << 16);
}
__device__ __forceinline__ uint4 rescale(uint4 q, float r) {
  if (is_power_of_two(r) && r >= 3.0517578125e-5f) {
    const __half2 h = __float2half2_rn(r);
    return make_uint4(rescale_word_half(q.x, h), rescale_word_half(q.y, h), rescale_word_half(q.z, h),
                      rescale_word_half(q.w, h));
  }
  return make_uint4(rescale_word(q.x, r), rescale_word(q.y, r), rescale_word(q.z, r), rescale_word(q.w, r));
}

// ------------------------------------------------------------------ append
struct AppendArgs {
  const void* x[2];            // k, v
  int64_t stride_t[2], stride_h[2];
  uint8_t* cache[2];
  int64_t stride_block[2], stride_row[2], stride_head[2];
  float* scale[2];
  const int32_t* cu;
  const int32_t* ctx;
  const int32_t* table;
  int64_t stride_table;
  int table_width, b, h_kv, num_blocks, page, page_shift, n;
};

// Index of the sequence that owns work item w, by a whole block: item bases
// f(i) grow with i, so it is the number of i in [1, b) with f(i) <= w.
template <typename F>
__device__ __forceinline__ int owner_of(int w, int b, F f) {
  int owner = 0;
  for (int i0 = 1; i0 < b; i0 += blockDim.x) {
    const int i = i0 + (int)threadIdx.x;
    const int c = __syncthreads_count(i < b && f(i) <= w);
    owner += c;
    if (c < (int)blockDim.x) break;
  }
  return owner;
}

// A task is one (sequence, block of the cache, head): its new rows of k and
// v are read once into registers (kVec 16-byte vectors of each per thread),
// their largest magnitudes give the two scales, and the quantised rows are
// written.  TEAM warps share a task.  Bound by its 3 bytes per element; a
// task of one token (a decode step) is one warp's, a block of a prompt is a
// whole team's so that its loads are all in flight together, and k and v
// share what finding the task costs (about 300 instructions, as many as
// quantising eight vectors).  A block of more rows than a team holds is read
// twice (the second time from L2).
//
// 16 prompts of 60 to 4,100 tokens, 8 heads, d = 128 (111 MB): 27 us, 4.1
// TB/s against 6.5 of a copy: 124 registers leave two CTAs to an SM, 4.2 waves
// of them that begin with a chain of dependent loads (offsets, block id, scale,
// row); the issue slots are half full.  256 tokens of as many sequences: 6.3
// us, that chain behind a launch.
//
// Which blocks a sequence touches is not known on the host.  Sequence i
// with n_i new tokens touches at most n_i / P + 2 blocks, so the items
// [cu_i / P + 2 i, cu_{i+1} / P + 2 (i + 1)) are enough for it, and every
// CTA finds its own without a scan.
template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(256) gqa_append_kernel(const AppendArgs a) {
  constexpr int kVec = TEAM == 1 ? 2 : 8;
  constexpr int kLanes = TEAM * 32;
  constexpr int kVecPerRow = D / 8;                   // 16-byte vectors per row
  constexpr int kRowsPerPass = kLanes / kVecPerRow;   // rows that a team covers per vector
  constexpr int kRowsHeld = kRowsPerPass * kVec;
  constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
  __shared__ float s_red[2][8];
  auto cu = [&](int i) { return min(max(__ldg(a.cu + i), 0), a.n); };
  const int w = blockIdx.x;
  const int seq = owner_of(w, a.b, [&](int i) { return (cu(i) >> a.page_shift) + 2 * i; });
  const int t0 = cu(seq), n_i = max(0, cu(seq + 1) - t0);
  const int ctx = max(__ldg(a.ctx + seq), 0);
  const int start = ctx - n_i;  // position of the first new token (< 0: the tokens before 0 are skipped)
  const int item = w - ((t0 >> a.page_shift) + 2 * seq);  // < 0: offsets that do not ascend
  const int pi = (max(start, 0) >> a.page_shift) + item;
  const int64_t pos0 = (int64_t)pi * a.page;
  if (n_i == 0 || item < 0 || pos0 >= ctx || pi >= a.table_width) return;
  const int blk = __ldg(a.table + (int64_t)seq * a.stride_table + pi);
  if (blk < 0 || blk >= a.num_blocks) return;

  const int team = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int head = blockIdx.y * (256 / kLanes) + team;
  const bool live = head < a.h_kv;  // teams past the last head only take part in the barriers
  const int first = max(start, (int)pos0), last = min((int64_t)ctx, pos0 + a.page);
  const int rows = live ? last - first : 0;
  const int r0 = first - (int)pos0;  // row in the block of the first new token
  const int old = start > pos0 ? r0 : 0;
  const int row = lane / kVecPerRow, col = lane % kVecPerRow;
  const int64_t token = t0 + first - start + row;
  const uint4* src[2];
  int64_t step[2];  // kRowsPerPass rows, in 16-byte vectors
  uint8_t* page[2];
  float* scale[2];
  float s_old[2] = {0.f, 0.f};
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    src[kv] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x[kv]) + token * a.stride_t[kv] +
                                             (int64_t)head * a.stride_h[kv]) + col;
    step[kv] = a.stride_t[kv] / 8 * kRowsPerPass;
    page[kv] = a.cache[kv] + (int64_t)blk * a.stride_block[kv] + (int64_t)head * a.stride_head[kv];
    scale[kv] = a.scale[kv] + (int64_t)blk * a.h_kv + head;
    if (old && live) s_old[kv] = *scale[kv];
  }

  uint4 x[2][kVec];
  auto load = [&](int base) {  // base: a multiple of kRowsHeld
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint4* p = src[kv] + (int64_t)(base / kRowsPerPass) * step[kv];
#pragma unroll
      for (int i = 0; i < kVec; ++i, p += step[kv])
        x[kv][i] = base + i * kRowsPerPass + row < rows ? __ldg(p) : make_uint4(0, 0, 0, 0);
    }
  };
  // The largest magnitudes: of the values' bits without signs, whose order
  // is the values', two at a time.  Infinities and NaN, which do not count,
  // are left out by a second look where there are any.
  uint32_t top[2] = {0, 0};
  for (int base = 0; base < rows; base += kRowsHeld) {
    load(base);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[kv][i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) t = max_halves(t, q[j] & 0x7FFF7FFFu);
      }
      if (max(t & 0xFFFFu, t >> 16) >= kInf) {
        t = 0;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[kv][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = q[j] & 0x7FFFu, hi = (q[j] >> 16) & 0x7FFFu;
            t = max(t, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
          }
        }
      }
      top[kv] = max(top[kv], max(t & 0xFFFFu, t >> 16));
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) top[kv] = __reduce_max_sync(0xffffffffu, top[kv]);
  float amax[2] = {to_f32x2<T>(top[0]).x, to_f32x2<T>(top[1]).x};
  if constexpr (TEAM > 1) {
    if ((threadIdx.x & 31) == 0) {
      s_red[0][threadIdx.x >> 5] = amax[0];
      s_red[1][threadIdx.x >> 5] = amax[1];
    }
    __syncthreads();  // also: every thread has read s_old before the scale is written
#pragma unroll
    for (int i = 0; i < TEAM; ++i) {
      amax[0] = fmaxf(amax[0], s_red[0][team * TEAM + i]);
      amax[1] = fmaxf(amax[1], s_red[1][team * TEAM + i]);
    }
  } else {
    __syncwarp();
  }
  if (!live) return;
  float s[2], inv[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    s[kv] = __uint_as_float((uint32_t)(scale_exponent(amax[kv]) + 127) << 23);
    if (old) s[kv] = fmaxf(s[kv], s_old[kv]);
    inv[kv] = 1.f / s[kv];
    if (lane == 0) *scale[kv] = s[kv];
    if (old && s[kv] != s_old[kv]) {
      const float ratio = s_old[kv] / s[kv];
      for (int e = lane; e < old * (D / 16); e += kLanes) {
        uint4* p = reinterpret_cast<uint4*>(page[kv] + (int64_t)(e / (D / 16)) * a.stride_row[kv]) + e % (D / 16);
        *p = rescale(*p, ratio);
      }
    }
  }
  for (int base = 0; base < rows; base += kRowsHeld) {
    if (rows > kRowsHeld) load(base);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      if (!is_power_of_two(s[kv])) continue;
      uint8_t* p = page[kv] + (int64_t)(r0 + base + row) * a.stride_row[kv] + col * 8;
      const int64_t next = a.stride_row[kv] * kRowsPerPass;
#pragma unroll
      for (int i = 0; i < kVec; ++i, p += next) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[kv][i]);
        if (base + i * kRowsPerPass + row < rows) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // a power of two divides exactly by its reciprocal
            const float2 f = scaled(to_f32x2<T>(q[j]), inv[kv]);
            b[j] = to_e4m3x2(f.x, f.y);
          }
          *reinterpret_cast<uint2*>(p) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
        }
      }
    }
  }
  // Another scale (a block that the caller filled by a rule of their own)
  // takes the division, which unrolled above would crowd out the rest.
#pragma unroll 1
  for (int kv = 0; kv < 2; ++kv) {
    const float sc = kv ? s[1] : s[0];
    if (is_power_of_two(sc)) continue;
#pragma unroll 1
    for (int r = row; r < rows; r += kRowsPerPass) {
      const uint4 v = __ldg((kv ? src[1] : src[0]) + (int64_t)(r / kRowsPerPass) * (kv ? step[1] : step[0]));
      const uint32_t q[4] = {v.x, v.y, v.z, v.w};
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = to_f32x2<T>(q[j]);
        b[j] = to_e4m3x2(f.x / sc, f.y / sc);
      }
      *reinterpret_cast<uint2*>((kv ? page[1] : page[0]) + (int64_t)(r0 + r) * (kv ? a.stride_row[1] : a.stride_row[0]) +
                                col * 8) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
    }
  }
}

template <typename T, int D>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
  const int items = a.n / a.page + 2 * a.b;
  // From about 8 tokens a sequence on, a block's rows fill a team of four
  // warps' registers; below it they are mostly one warp's.
  if (a.n > 8 * (int64_t)a.b)
    gqa_append_kernel<T, D, 4><<<dim3(items, (a.h_kv + 1) / 2), 256, 0, stream>>>(a);
  else
    gqa_append_kernel<T, D, 1><<<dim3(items, (a.h_kv + 7) / 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ eviction
struct EvictArgs {
  int budget, recent, width, new_width, page, page_shift, table_width, new_table_width, num_blocks, h_kv, b;
  const float* weights;
  int64_t stride_w_b, stride_w_h;
  float* new_weights;
  int64_t stride_nw_b, stride_nw_h;
  int32_t* kept;
  int32_t* new_lens;
  const int32_t* table;
  int64_t stride_table;
  const int32_t* new_table;
  int64_t stride_new_table;
  const int32_t* ctx;
  uint8_t* cache[2];
  int64_t stride_block[2], stride_row[2], stride_head[2];
  float* scale[2];
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int seq) {
  const int64_t room = min((int64_t)a.table_width * a.page, (int64_t)a.width);
  return (int)min((int64_t)max(__ldg(a.ctx + seq), 0), room);
}

// Bits whose unsigned order is the order of the weights: NaN above all
// numbers, +0 and -0 alike.  Adding zero makes -0 +0 and any NaN the one
// with all bits but the sign set.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t bits = __float_as_uint(__fadd_rn(w, 0.f));
  return bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u);
}

constexpr int kSelThreads = 1024;
constexpr int kChunk = 4 * kSelThreads;  // positions of a step, four to a thread
constexpr int kBins = 2048;              // digits of 11, 11 and 10 bits
constexpr int kHists = 4;                // copies of the histogram, against conflicts on near weights
constexpr int kList = 3400;              // keys of one digit that are listed (static shared memory ends at 48 KB)

// One CTA per (sequence, KV head): the key of the last position that is kept
// by a radix histogram from the top digit down, then one ordered pass that
// writes the kept positions (a running count of those above that key and of
// those equal to it; of the latter only the first ones are kept).  Where few
// keys share the top digit (a digit of sign, exponent and two bits spreads
// weights of one magnitude over some bins), they are listed and the other
// digits look at the list only, so the weights are read three times (from L2
// after the first).  Exact zeros, of positions that nothing looked at, are
// counted by vote instead of by conflicting atomics.  Bound by instructions
// (65 % of the issue slots), and by the longest sequence.  32 sequences of
// up to 32,768, 8 heads: 31 us; an earlier form with the keys held in
// registers and one CTA per SM 37, with 512 threads 45, with a cluster of
// four CTAs per sequence that sum their histograms over distributed shared
// memory 66 (its fixed cost, paid four times, outweighs the split).
__global__ void __launch_bounds__(kSelThreads, 2) gqa_evict_select_kernel(const EvictArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ alignas(16) uint32_t hist[kHists][kBins];
  __shared__ uint32_t list[kList];
  __shared__ uint32_t s_scan[kSelThreads / 32];
  __shared__ uint32_t s_prefix, s_found;
  __shared__ int s_need, s_count;
  const int head = blockIdx.x, seq = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = evict_len(a, seq);
  const int new_len = min(len, a.budget);
  const float* w = a.weights + (int64_t)seq * a.stride_w_b + (int64_t)head * a.stride_w_h;
  float* nw = a.new_weights + (int64_t)seq * a.stride_nw_b + (int64_t)head * a.stride_nw_h;
  int32_t* kept = a.kept + ((int64_t)seq * a.h_kv + head) * a.budget;
  const int recent = len > a.budget ? a.recent : len;  // positions that are kept without a look
  const int older = len - recent;
  const int pick = new_len - recent;  // of the older ones
  if (head == 0 && tid == 0) a.new_lens[seq] = new_len;
  for (int i = new_len + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  for (int i = new_len + tid; i < a.new_width; i += kSelThreads) nw[i] = 0.f;
  for (int i = tid; i < recent; i += kSelThreads) {
    kept[new_len - recent + i] = older + i;
    nw[new_len - recent + i] = __ldg(w + older + i);
  }
  if (pick == 0) return;
  // f(i, keys, weights) for each four positions from i on; those that are not
  // older ones have the key 0, which no weight's is
  const bool vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  auto four = [&](int i, auto f) {
    if (vec && i + 4 <= older) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(w + i));
      const float v[4] = {x.x, x.y, x.z, x.w};
      const uint32_t k[4] = {weight_key(x.x), weight_key(x.y), weight_key(x.z), weight_key(x.w)};
      f(k, v);
    } else {
      float v[4];
      uint32_t k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = i + j < older ? __ldg(w + i + j) : 0.f;
        k[j] = i + j < older ? weight_key(v[j]) : 0u;
      }
      f(k, v);
    }
  };

  constexpr uint32_t kZero = 0x80000000u;  // weight_key(0)
  bool listed = false;
  uint32_t prefix = 0;
  int need = pick, same = 0;  // the need-th largest key is looked for among those that share `prefix`, `same` of them
  // One digit: count(histogram) adds the keys with the prefix to the copies
  // and returns how many zeros there are among them, which it leaves out.
  auto digit = [&](int shift, int bits, auto count) {
    for (int i = 4 * tid; i < kHists * kBins; i += 4 * kSelThreads)
      *reinterpret_cast<uint4*>(&hist[0][0] + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const uint32_t zeros = __reduce_add_sync(0xffffffffu, count(hist[(tid >> 1) % kHists]));
    if (lane == 0 && zeros) atomicAdd(&hist[0][(kZero >> shift) & ((1u << bits) - 1)], zeros);
    __syncthreads();
    // thread t has the two bins below 2048 - 2 t, the largest keys first
    const int bin0 = kBins - 2 * (tid + 1);
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kHists; ++k) {
      const uint2 v = *reinterpret_cast<const uint2*>(&hist[k][bin0]);
      c[0] += v.y;
      c[1] += v.x;
    }
    uint32_t incl = c[0] + c[1], before = 0u - incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    before += incl + __reduce_add_sync(0xffffffffu, lane < warp ? s_scan[lane] : 0u);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if ((int)before < need && need <= (int)(before + c[j])) {
        s_prefix = (prefix << bits) | (uint32_t)(bin0 + 1 - j);
        s_need = need - (int)before;
        s_count = (int)c[j];
      }
      before += c[j];
    }
    if (tid == 0 && !listed) s_found = 0;
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    same = s_count;
  };
  digit(21, 11, [&](uint32_t* h) {
    uint32_t zeros = 0;
#pragma unroll 2
    for (int i = 4 * tid; i < older; i += kChunk)
      four(i, [&](const uint32_t(&k)[4], const float(&)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (k[j] == kZero) ++zeros;
          else if (k[j] != 0) atomicAdd(&h[k[j] >> 21], 1u);
        }
      });
    return zeros;
  });
  if (same <= kList) {
    listed = true;
#pragma unroll 2
    for (int i = 4 * tid; i < older; i += kChunk)
      four(i, [&](const uint32_t(&k)[4], const float(&)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((k[j] >> 21) == prefix) list[atomicAdd(&s_found, 1u)] = k[j];
      });
  }
#pragma unroll 1
  for (int shift = 10; shift >= 0; shift -= 10) {
    const int bits = shift ? 11 : 10;
    digit(shift, bits, [&](uint32_t* h) {
      uint32_t zeros = 0;
      auto one = [&](uint32_t k) {
        if ((k >> shift >> bits) != prefix || k == 0) return;
        if (k == kZero) ++zeros;
        else atomicAdd(&h[(k >> shift) & ((1u << bits) - 1)], 1u);
      };
      if (listed) {
        for (int i = tid; i < (int)s_found; i += kSelThreads) one(list[i]);
      } else {
#pragma unroll 1
        for (int i = 4 * tid; i < older; i += kChunk)
          four(i, [&](const uint32_t(&k)[4], const float(&)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) one(k[j]);
          });
      }
      return zeros;
    });
  }

  // prefix is the last kept key; `need` of the `same` positions equal to it
  // are kept: mostly all of them, otherwise the first.  Counts of those kept
  // for certain (the low half of a step's sum) and of those equal (the high).
  const bool ties = need < same, top = ties && prefix == 0xFFFFFFFFu;  // top: nothing lies above the last key
  const uint32_t sure = ties && !top ? prefix + 1 : prefix;
  uint32_t above = 0, equal = 0;  // counts before this step
#pragma unroll 1
  for (int base = 0; base < older; base += kChunk) {
    const int i = base + 4 * tid;
    uint32_t k[4];
    float v[4];
    four(i, [&](const uint32_t(&kk)[4], const float(&vv)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[j] = kk[j];
        v[j] = vv[j];
      }
    });
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) n += k[j] >= sure && !top ? 1u : 0u;
    if (ties) {
#pragma unroll
      for (int j = 0; j < 4; ++j) n += k[j] == prefix ? 1u << 16 : 0u;
    }
    uint32_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    const uint32_t sums = s_scan[lane];
    const uint32_t pre = __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0u) + incl - n;
    const uint32_t total = __reduce_add_sync(0xffffffffu, sums);
    __syncthreads();  // s_scan is read
    uint32_t g = above + (pre & 0xFFFFu), e = equal + (pre >> 16);
    if (!ties) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (k[j] >= sure) {
          kept[g] = i + j;
          nw[g] = v[j];
          ++g;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool is_above = k[j] >= sure && !top, is_equal = k[j] == prefix;
        if (is_above || (is_equal && e < (uint32_t)need)) {
          const uint32_t at = g + min(e, (uint32_t)need);
          kept[at] = i + j;
          nw[at] = v[j];
        }
        g += is_above;
        e += is_equal;
      }
    }
    above += total & 0xFFFFu;
    equal += total >> 16;
  }
}

// One CTA per (new block, KV head, sequence): the sources of its rows, then
// the rows of K and V, 16 bytes per thread and load, and, while those are on
// their way, the largest of the sources' scales.  Bound by the kept bytes,
// read (rows at random places) and written once: with the selection, 4,096
// of up to 32,768 positions of 32 sequences, 8 heads (560 MB in all) take 129
// us, 97 of them here, 5.5 TB/s; 2,048 of 8,192 of one sequence 14.5 us, two
// launches' and chains' latency.
constexpr int kGatherThreads = 128;
struct Source {
  int64_t off;  // bytes, -1: nothing there
  float scale;
  int unused;
};
template <int D>
__global__ void __launch_bounds__(kGatherThreads, 8) gqa_evict_gather_kernel(const EvictArgs a) {
  constexpr int kVec = D / 16;
  constexpr int kUnroll = 4;  // of K and of V: all of 64 rows of 128 in flight at once
  extern __shared__ Source s_src[];  // [2][page]
  __shared__ float s_red[2][kGatherThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the kept positions
  const int nb = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
  const int len = evict_len(a, seq);
  const int new_len = min(len, a.budget);
  const int j0 = nb * a.page;
  if (j0 >= new_len || nb >= a.new_table_width) return;
  const int dest = __ldg(a.new_table + (int64_t)seq * a.stride_new_table + nb);
  if (dest < 0 || dest >= a.num_blocks) return;
  const int rows = min(a.page, new_len - j0);
  const int32_t* kept = a.kept + ((int64_t)seq * a.h_kv + head) * a.budget + j0;
  float top[2] = {0.f, 0.f}, mine[2] = {0.f, 0.f};  // mine: of row tid, not looked at before the loads below
  for (int r = tid; r < rows; r += kGatherThreads) {
    const int t = kept[r];
    const int blk = t >= 0 && t < len ? __ldg(a.table + (int64_t)seq * a.stride_table + (t >> a.page_shift)) : -1;
    const bool ok = blk >= 0 && blk < a.num_blocks;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float scale = ok ? a.scale[kv][(int64_t)blk * a.h_kv + head] : 0.f;
      s_src[kv * a.page + r].off = ok ? (int64_t)blk * a.stride_block[kv] + (int64_t)(t & (a.page - 1)) * a.stride_row[kv] +
                                            (int64_t)head * a.stride_head[kv]
                                      : -1;
      if (r < kGatherThreads) {
        mine[kv] = scale;
      } else {
        s_src[kv * a.page + r].scale = scale;
        top[kv] = fmaxf(top[kv], scale);
      }
    }
  }
  __syncthreads();
  const int n = rows * kVec;
  uint8_t* to[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    to[kv] = a.cache[kv] + (int64_t)dest * a.stride_block[kv] + (int64_t)head * a.stride_head[kv] + tid % kVec * 16;
  static_assert(kGatherThreads % kVec == 0, "a thread keeps its 16 bytes of a row");
  uint4 q[2][kUnroll];
  auto load = [&](int e0) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int e = e0 + u * kGatherThreads;
        q[kv][u] = make_uint4(0, 0, 0, 0);
        if (e < n) {
          const int64_t off = s_src[kv * a.page + e / kVec].off;
          if (off >= 0) q[kv][u] = *reinterpret_cast<const uint4*>(a.cache[kv] + off + tid % kVec * 16);
        }
      }
  };
  load(tid);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    if (tid < rows) s_src[kv * a.page + tid].scale = mine[kv];
    top[kv] = fmaxf(top[kv], mine[kv]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top[kv] = fmaxf(top[kv], __shfl_xor_sync(0xffffffffu, top[kv], o));
    if ((tid & 31) == 0) s_red[kv][tid >> 5] = top[kv];
  }
  __syncthreads();
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
    for (int i = 0; i < kGatherThreads / 32; ++i) top[kv] = fmaxf(top[kv], s_red[kv][i]);
    if (tid == 0) a.scale[kv][(int64_t)dest * a.h_kv + head] = top[kv];
  }
  for (int e0 = tid; e0 < n; e0 += kGatherThreads * kUnroll) {
    if (e0 != tid) load(e0);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int e = e0 + u * kGatherThreads;
        if (e < n) {
          const float scale = s_src[kv * a.page + e / kVec].scale;
          if (scale != top[kv]) q[kv][u] = rescale(q[kv][u], scale / top[kv]);  // 0 <= scale < top
          *reinterpret_cast<uint4*>(to[kv] + (int64_t)(e / kVec) * a.stride_row[kv]) = q[kv][u];
        }
      }
  }
}

}  // namespace

cudaError_t launch_gqa_append(const dsv4b_gqa_cache& c, int dtype, const void* k, int64_t stride_k_t,
                              int64_t stride_k_h, const void* v, int64_t stride_v_t, int64_t stride_v_h,
                              const int32_t* cu_seqlens, int n, cudaStream_t stream) {
  AppendArgs a = {};
  a.x[0] = k;
  a.x[1] = v;
  a.stride_t[0] = stride_k_t;
  a.stride_t[1] = stride_v_t;
  a.stride_h[0] = stride_k_h;
  a.stride_h[1] = stride_v_h;
  a.cache[0] = static_cast<uint8_t*>(c.k);
  a.cache[1] = static_cast<uint8_t*>(c.v);
  a.stride_block[0] = c.stride_k_block;
  a.stride_block[1] = c.stride_v_block;
  a.stride_row[0] = c.stride_k_row;
  a.stride_row[1] = c.stride_v_row;
  a.stride_head[0] = c.stride_k_head;
  a.stride_head[1] = c.stride_v_head;
  a.scale[0] = c.k_scale;
  a.scale[1] = c.v_scale;
  a.cu = cu_seqlens;
  a.ctx = c.context_lens;
  a.table = c.block_table;
  a.stride_table = c.stride_block_table;
  a.table_width = c.table_width;
  a.b = c.b;
  a.h_kv = c.h_kv;
  a.num_blocks = c.num_blocks;
  a.page = c.page_block_size;
  while ((1 << a.page_shift) < a.page) ++a.page_shift;
  a.n = n;
  if (dtype == DSV4B_BF16)
    return c.d == 128 ? launch_append<__nv_bfloat16, 128>(a, stream) : launch_append<__nv_bfloat16, 64>(a, stream);
  return c.d == 128 ? launch_append<__half, 128>(a, stream) : launch_append<__half, 64>(a, stream);
}

cudaError_t launch_gqa_evict(const dsv4b_gqa_cache& c, const dsv4b_gqa_evict_params& e, cudaStream_t stream) {
  EvictArgs a = {};
  a.budget = e.budget;
  a.recent = e.recent;
  a.width = e.width;
  a.new_width = e.new_width;
  a.page = c.page_block_size;
  while ((1 << a.page_shift) < a.page) ++a.page_shift;
  a.table_width = c.table_width;
  a.new_table_width = e.new_table_width;
  a.num_blocks = c.num_blocks;
  a.h_kv = c.h_kv;
  a.b = c.b;
  a.weights = e.weights;
  a.stride_w_b = e.stride_w_b;
  a.stride_w_h = e.stride_w_h;
  a.new_weights = e.new_weights;
  a.stride_nw_b = e.stride_nw_b;
  a.stride_nw_h = e.stride_nw_h;
  a.kept = e.kept;
  a.new_lens = e.new_lens;
  a.table = c.block_table;
  a.stride_table = c.stride_block_table;
  a.new_table = e.new_table;
  a.stride_new_table = e.stride_new_table;
  a.ctx = c.context_lens;
  a.cache[0] = static_cast<uint8_t*>(c.k);
  a.cache[1] = static_cast<uint8_t*>(c.v);
  a.stride_block[0] = c.stride_k_block;
  a.stride_block[1] = c.stride_v_block;
  a.stride_row[0] = c.stride_k_row;
  a.stride_row[1] = c.stride_v_row;
  a.stride_head[0] = c.stride_k_head;
  a.stride_head[1] = c.stride_v_head;
  a.scale[0] = c.k_scale;
  a.scale[1] = c.v_scale;
  gqa_evict_select_kernel<<<dim3(c.h_kv, c.b), kSelThreads, 0, stream>>>(a);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const int blocks = (int)(((int64_t)e.budget + c.page_block_size - 1) / c.page_block_size);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks < e.new_table_width ? blocks : e.new_table_width, c.h_kv, c.b);
  cfg.blockDim = dim3(kGatherThreads);
  cfg.dynamicSmemBytes = (size_t)c.page_block_size * 2 * sizeof(Source);  // <= 32 KB
  cfg.stream = stream;
  cudaLaunchAttribute attr;  // starts while the selection ends; waits for it in the kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return c.d == 128 ? cudaLaunchKernelEx(&cfg, gqa_evict_gather_kernel<128>, a)
                    : cudaLaunchKernelEx(&cfg, gqa_evict_gather_kernel<64>, a);
}

}  // namespace dsv4b
