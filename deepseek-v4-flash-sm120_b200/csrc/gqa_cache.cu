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
// Four e4m3 of a word times r, rounded again.
__device__ __forceinline__ uint32_t rescale_word(uint32_t w, float r) {
  const float2 a = scaled(from_e4m3x2(w & 0xFFFFu), r), b = scaled(from_e4m3x2(w >> 16), r);
  return to_e4m3x2(a.x, a.y) | (to_e4m3x2(b.x, b.y) << 16);
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

// A task is one (sequence, block of the cache, head, k or v): its new rows
// are read once into registers (kVec 16-byte vectors per thread), their
// largest magnitude gives the scale, and the quantised rows are written.
// TEAM warps share a task.  Bound by its 3 bytes per element; a task of one
// token (a decode step) is one warp's, a page of a prompt is a whole team's
// so that its loads are all in flight together.  A block of more rows than
// a team holds is read twice (the second time from L2).
//
// Which blocks a sequence touches is not known on the host.  Sequence i
// with n_i new tokens touches at most n_i / P + 2 blocks, so the items
// [cu_i / P + 2 i, cu_{i+1} / P + 2 (i + 1)) are enough for it, and every
// CTA finds its own without a scan.
template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(256) gqa_append_kernel(const AppendArgs a) {
  constexpr int kVec = 8;
  constexpr int kLanes = TEAM * 32;
  constexpr int kVecPerRow = D / 8;                   // 16-byte vectors per row
  constexpr int kRowsPerPass = kLanes / kVecPerRow;   // rows that a team covers per vector
  constexpr int kRowsHeld = kRowsPerPass * kVec;
  __shared__ float s_red[8];
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
  const int task = blockIdx.y * (256 / kLanes) + team;
  const bool live = task < 2 * a.h_kv;  // teams past the last task only take part in the barriers
  const int kv = live ? task / a.h_kv : 0, head = live ? task % a.h_kv : 0;
  const int first = max(start, (int)pos0), last = min((int64_t)ctx, pos0 + a.page);
  const int rows = live ? last - first : 0;
  const int r0 = first - (int)pos0;  // row in the block of the first new token
  const int old = start > pos0 ? start - (int)pos0 : 0;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x[kv]) +
                                                    (int64_t)(t0 + first - start) * a.stride_t[kv] +
                                                    (int64_t)head * a.stride_h[kv]) + lane % kVecPerRow;
  const int64_t step = a.stride_t[kv] / 8;  // in 16-byte vectors
  const int row = lane / kVecPerRow;
  uint8_t* page = a.cache[kv] + (int64_t)blk * a.stride_block[kv] + (int64_t)head * a.stride_head[kv];
  float* scale = a.scale[kv] + (int64_t)blk * a.h_kv + head;
  const float s_old = old && live ? *scale : 0.f;

  uint4 x[kVec];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int r = base + i * kRowsPerPass + row;
      x[i] = r < rows ? __ldg(src + r * step) : make_uint4(0, 0, 0, 0);
    }
  };
  // The largest magnitude: of the values' bits without signs, whose order is
  // the values', two at a time.  Infinities and NaN, which do not count, are
  // left out by a second look where there are any.
  constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
  uint32_t top = 0;
  for (int base = 0; base < rows; base += kRowsHeld) {
    load(base);
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) t = max_halves(t, q[j] & 0x7FFF7FFFu);
    }
    if (max(t & 0xFFFFu, t >> 16) >= kInf) {
      t = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = q[j] & 0x7FFFu, hi = (q[j] >> 16) & 0x7FFFu;
          t = max(t, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
        }
      }
    }
    top = max(top, max(t & 0xFFFFu, t >> 16));
  }
  float amax = to_f32x2<T>(top).x;
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (TEAM > 1) {
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = amax;
    __syncthreads();  // also: every thread has read s_old before the scale is written
#pragma unroll
    for (int i = 0; i < TEAM; ++i) amax = fmaxf(amax, s_red[team * TEAM + i]);
  } else {
    __syncwarp();
  }
  if (!live) return;
  float s = __uint_as_float((uint32_t)(scale_exponent(amax) + 127) << 23);
  if (old) s = fmaxf(s, s_old);
  if (lane == 0) *scale = s;
  if (old && s != s_old) {
    const float ratio = s_old / s;
    for (int e = lane; e < old * (D / 16); e += kLanes) {
      uint4* p = reinterpret_cast<uint4*>(page + (int64_t)(e / (D / 16)) * a.stride_row[kv]) + e % (D / 16);
      uint4 q = *p;
      q.x = rescale_word(q.x, ratio);
      q.y = rescale_word(q.y, ratio);
      q.z = rescale_word(q.z, ratio);
      q.w = rescale_word(q.w, ratio);
      *p = q;
    }
  }
  // A power of two divides exactly by its reciprocal; any other scale (a
  // block that the caller filled by a rule of their own) takes the division.
  const bool exact = is_power_of_two(s);
  const float inv = 1.f / s;
  for (int base = 0; base < rows; base += kRowsHeld) {
    if (rows > kRowsHeld) load(base);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int r = base + i * kRowsPerPass + row;
      if (r < rows) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[i]);
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 f = to_f32x2<T>(q[j]);
          if (exact) {
            f = scaled(f, inv);
          } else {
            f.x /= s;
            f.y /= s;
          }
          b[j] = to_e4m3x2(f.x, f.y);
        }
        *reinterpret_cast<uint2*>(page + (int64_t)(r0 + r) * a.stride_row[kv] + (lane % kVecPerRow) * 8) =
            make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
  const int items = a.n / a.page + 2 * a.b;
  // From about 8 tokens a sequence on, a block's rows fill a team of four
  // warps' registers; below it they are mostly one warp's.
  if (a.n > 8 * (int64_t)a.b)
    gqa_append_kernel<T, D, 4><<<dim3(items, (2 * a.h_kv + 1) / 2), 256, 0, stream>>>(a);
  else
    gqa_append_kernel<T, D, 1><<<dim3(items, (2 * a.h_kv + 7) / 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ eviction
struct EvictArgs {
  int budget, recent, width, new_width, page, table_width, new_table_width, num_blocks, h_kv, b;
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
// numbers, +0 and -0 alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t bits = __float_as_uint(w + 0.f);  // -0 + 0 = +0
  return bits ^ ((bits >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr int kSelThreads = 1024;
constexpr int kChunk = 4 * kSelThreads;  // positions of a step, four to a thread
constexpr int kHeld = 8;                 // steps whose keys a thread keeps: 32,768 positions
constexpr int kBins = 2048;              // digits of 11, 11 and 10 bits
constexpr int kHists = 4;                // copies of the histogram, against conflicts on near weights

// One CTA per (sequence, KV head): the key of the last position that is kept
// by three passes of a radix histogram from the top digit down, then one
// ordered pass that writes the kept positions (a running count of those
// above that key and of those equal to it; of the latter only the first ones
// are kept).  The weights are read once into registers (32 a thread; longer
// sequences are read again, from L2, in every pass).  The histogram's
// conflicts bound it: a digit of sign, exponent and two bits spreads weights
// of one magnitude over some bins, and exact zeros (positions that nothing
// looked at) are counted by vote.
__global__ void __launch_bounds__(kSelThreads) gqa_evict_select_kernel(const EvictArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ uint32_t hist[kHists][kBins];
  __shared__ uint32_t s_scan[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = evict_len(a, seq);
  const int new_len = min(len, a.budget);
  const float* w = a.weights + (int64_t)seq * a.stride_w_b + (int64_t)head * a.stride_w_h;
  float* nw = a.new_weights + (int64_t)seq * a.stride_nw_b + (int64_t)head * a.stride_nw_h;
  int32_t* kept = a.kept + ((int64_t)seq * a.h_kv + head) * a.budget;
  if (head == 0 && tid == 0) a.new_lens[seq] = new_len;
  const int recent = len > a.budget ? a.recent : len;  // positions that are kept without a look
  const int older = len - recent;
  const int pick = new_len - recent;  // of the older ones
  // four positions from i on, as keys; those that are not older ones are 0,
  // which no weight's key is
  const bool vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  auto keys_at = [&](int i, uint32_t (&k)[4]) {
    float x[4];
    if (vec && i + 4 <= older) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(w + i));
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = i + j < older ? __ldg(w + i + j) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = i + j < older ? weight_key(x[j]) : 0u;
  };
  const bool held = older <= kHeld * kChunk;
  uint32_t mine[kHeld][4];
  if (pick > 0 && held) {
#pragma unroll
    for (int s = 0; s < kHeld; ++s) keys_at(s * kChunk + 4 * tid, mine[s]);
  }
  for (int i = new_len + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  for (int i = new_len + tid; i < a.new_width; i += kSelThreads) nw[i] = 0.f;
  for (int i = tid; i < recent; i += kSelThreads) {
    kept[new_len - recent + i] = older + i;
    nw[new_len - recent + i] = __ldg(w + older + i);
  }
  if (pick == 0) return;
  // f(step, keys) over all steps
  auto each = [&](auto f) {
    if (held) {
#pragma unroll
      for (int s = 0; s < kHeld; ++s)
        if (s * kChunk < older) f(s, mine[s]);
    } else {
      for (int s = 0; s * kChunk < older; ++s) {
        uint32_t k[4];
        keys_at(s * kChunk + 4 * tid, k);
        f(s, k);
      }
    }
  };

  constexpr uint32_t kZero = 0x80000000u;  // weight_key(0)
  uint32_t prefix = 0;
  int need = pick;  // the need-th largest key is looked for among those that share `prefix`
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kHists * kBins; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    uint32_t* h = hist[(tid >> 1) % kHists];
    uint32_t zeros = 0;
    each([&](int, const uint32_t(&k)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = k[j] != 0 && (pass == 0 || (k[j] >> (shift + bits)) == prefix);
        if (in && k[j] == kZero) ++zeros;
        if (in && k[j] != kZero) atomicAdd(&h[(k[j] >> shift) & ((1u << bits) - 1)], 1u);
      }
    });
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (lane == 0 && zeros) atomicAdd(&hist[0][(kZero >> shift) & ((1u << bits) - 1)], zeros);
    __syncthreads();
    // thread t has the two bins below 2048 - 2 t, the largest keys first
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < kHists; ++k) c[j] += hist[k][kBins - 1 - (2 * tid + j)];
    uint32_t incl = c[0] + c[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    const uint32_t others = __reduce_add_sync(0xffffffffu, lane < warp ? s_scan[lane] : 0u);
    uint32_t before = others + incl - c[0] - c[1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if ((int)before < need && need <= (int)(before + c[j])) {
        s_prefix = (prefix << bits) | (uint32_t)(kBins - 1 - (2 * tid + j));
        s_need = need - (int)before;
      }
      before += c[j];
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // prefix is the last kept key; `need` of the positions equal to it are kept
  uint32_t above = 0, equal = 0;  // counts before this step
  each([&](int s, const uint32_t(&k)[4]) {
    uint32_t n = 0;  // (above << 16) | equal: a step has 4,096 positions
#pragma unroll
    for (int j = 0; j < 4; ++j) n += k[j] > prefix ? 1u << 16 : k[j] == prefix ? 1u : 0u;
    uint32_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    const uint32_t sums = s_scan[lane];
    const uint32_t pre = __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0u) + incl - n;
    const uint32_t total = __reduce_add_sync(0xffffffffu, sums);
    uint32_t g = above + (pre >> 16), e = equal + (pre & 0xFFFFu);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool is_above = k[j] > prefix, is_equal = k[j] == prefix;
      if (is_above || (is_equal && e < (uint32_t)need)) {
        const uint32_t at = g + min(e, (uint32_t)need);
        const int pos = s * kChunk + 4 * tid + j;
        kept[at] = pos;
        nw[at] = __ldg(w + pos);  // the weight itself: a key does not tell -0 from 0, nor NaN from NaN
      }
      g += is_above;
      e += is_equal;
    }
    above += total >> 16;
    equal += total & 0xFFFFu;
  });
}

// One CTA per (new block, KV head, sequence): the sources of its rows, the
// largest of their scales, then the rows of K and V, 16 bytes per thread
// and load.  Bound by the kept bytes, read and written once.
constexpr int kGatherThreads = 128;
template <int D>
__global__ void __launch_bounds__(kGatherThreads) gqa_evict_gather_kernel(const EvictArgs a) {
  constexpr int kVec = D / 16;
  constexpr int kUnroll = 8;  // K and V of 64 rows of 128: all loads in flight at once
  extern __shared__ uint8_t smem_raw[];
  int64_t* s_off = reinterpret_cast<int64_t*>(smem_raw);        // [2][page] source bytes, -1: nothing there
  float* s_scale = reinterpret_cast<float*>(s_off + 2 * a.page);  // [2][page]
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
  float top[2] = {0.f, 0.f};
  for (int r = tid; r < rows; r += kGatherThreads) {
    const int t = kept[r];
    const int blk = t >= 0 && t < len ? __ldg(a.table + (int64_t)seq * a.stride_table + t / a.page) : -1;
    const bool ok = blk >= 0 && blk < a.num_blocks;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float s = ok ? a.scale[kv][(int64_t)blk * a.h_kv + head] : 0.f;
      s_off[kv * a.page + r] = ok ? (int64_t)blk * a.stride_block[kv] + (int64_t)(t % a.page) * a.stride_row[kv] +
                                        (int64_t)head * a.stride_head[kv]
                                  : -1;
      s_scale[kv * a.page + r] = s;
      top[kv] = fmaxf(top[kv], s);
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
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
  // K's rows, then V's
  for (int e0 = tid; e0 < 2 * rows * kVec; e0 += kGatherThreads * kUnroll) {
    uint4 q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + u * kGatherThreads;
      q[u] = make_uint4(0, 0, 0, 0);
      if (e < 2 * rows * kVec) {
        const int kv = e >= rows * kVec, r = e / kVec - kv * rows;
        const int64_t off = s_off[kv * a.page + r];
        if (off >= 0) q[u] = *(reinterpret_cast<const uint4*>(a.cache[kv] + off) + e % kVec);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + u * kGatherThreads;
      if (e < 2 * rows * kVec) {
        const int kv = e >= rows * kVec, r = e / kVec - kv * rows;
        const float s = s_scale[kv * a.page + r];
        if (s != top[kv]) {
          const float ratio = s / top[kv];  // 0 <= s < top
          q[u].x = rescale_word(q[u].x, ratio);
          q[u].y = rescale_word(q[u].y, ratio);
          q[u].z = rescale_word(q[u].z, ratio);
          q[u].w = rescale_word(q[u].w, ratio);
        }
        uint8_t* to = a.cache[kv] + (int64_t)dest * a.stride_block[kv] + (int64_t)head * a.stride_head[kv];
        *(reinterpret_cast<uint4*>(to + (int64_t)r * a.stride_row[kv]) + e % kVec) = q[u];
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
  cfg.dynamicSmemBytes = (size_t)c.page_block_size * 24;  // <= 24 KB
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
