// The 8-bit KV cache in blocks: quantising write, read-back and eviction.
//
// A block holds B tokens (32, 64 or 128) of one sequence; per (block, kv
// head) K is [B, hd] int8, V is [hd, B] int8, each with one fp32 scale
// (mlb_ops.h).  Writing n new rows behind e earlier ones of a block:
//   s' = max(s if e > 0, amax(new) / 127)
//   new code = round(x / s'), earlier code = round(c s / s')
// Both quotients are rounded as if they were exact, so the codes depend on
// nothing but the definition.
#include <climits>
#include <cstdint>

#include "common.cuh"

namespace mlb {
namespace {

constexpr int kKv8Threads = 256;

// What a CTA works on: columns of the table that the rows of packed
// sequences touch, counted through all sequences.
struct Kv8Rows {
  const int32_t* table;
  const int32_t* offsets;
  const int32_t* positions;
  int64_t table_cols;
  int64_t n_blocks;
  int64_t rows;
  int n_seqs;
  int block;   // tokens per block
  int kv_heads;
  int hd;
  int32_t* status;
};

struct Kv8Span {
  int64_t row;     // packed row of the first token
  int64_t block;   // block id, -1: outside the table or a bad id
  int first;       // place of the first token in the block
  int count;       // tokens (0: nothing to do)
};

__device__ __forceinline__ void Raise(int32_t* status, int bits) {
  if (status != nullptr) atomicOr(status, bits);
}

// The index-th touched block over all sequences.  All threads of the CTA
// call it; every thread receives the span.  Sequences are scanned
// kKv8Threads at a time.
__device__ Kv8Span FindSpan(const Kv8Rows& a, int64_t index) {
  __shared__ int64_t warp_sum[kKv8Threads / 32];
  __shared__ Kv8Span found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) found = Kv8Span{0, -1, 0, 0};
  int64_t before = 0;
  for (int base = 0; base < a.n_seqs; base += kKv8Threads) {
    const int i = base + static_cast<int>(threadIdx.x);
    int64_t touched = 0, begin = 0, end = 0, position = 0;
    bool lost = false;
    if (i < a.n_seqs) {
      begin = a.offsets[i];
      end = a.offsets[i + 1];
      position = a.positions[i];
      lost = position < 0;  // its rows have no place: counted from 0, in no block
      if (lost) position = 0;
      if (begin < 0 || end < begin || end > a.rows) {
        if (index == 0) Raise(a.status, MLB_STATUS_BAD_LENGTH);
      } else if (end > begin) {
        touched = (position + end - begin - 1) / a.block - position / a.block + 1;
        if (lost && index == 0) Raise(a.status, MLB_STATUS_BAD_POSITION);
      }
    }
    int64_t sum = touched;  // inclusive scan over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kKv8Threads / 32; ++w) {
      if (w < warp) sum += warp_sum[w];
      total += warp_sum[w];
    }
    const int64_t local = index - (before + sum - touched);
    if (touched > 0 && local >= 0 && local < touched) {
      const int64_t col = position / a.block + local;
      const int64_t t0 = local == 0 ? position : col * a.block;
      const int64_t t1 = min(position + end - begin, (col + 1) * a.block);
      Kv8Span s;
      s.row = begin + t0 - position;
      s.first = static_cast<int>(t0 - col * a.block);
      s.count = static_cast<int>(t1 - t0);
      s.block = -1;
      if (col >= a.table_cols) {
        Raise(a.status, MLB_STATUS_BAD_POSITION);
      } else if (!lost) {
        const int32_t id = a.table[i * a.table_cols + col];
        if (id < 0 || id >= a.n_blocks)
          Raise(a.status, MLB_STATUS_BAD_BLOCK);
        else
          s.block = id;
      }
      found = s;
    }
    before += total;
    __syncthreads();
    if (index < before && index != 0) break;  // index 0 looks at every sequence's range
  }
  return found;
}

// round(x / s) as if the quotient were exact, clamped to [-127, 127]; inv is
// 1 / s.  r, the rounded approximate quotient, is off by at most one; the
// remainder x - r s is a multiple of the last place of s (or of x, for
// |r| <= 1) below 2 s, so the fused multiply-add gives it without error.
__device__ __forceinline__ int Quantise(float x, float s, float inv) {
  // 1 / s of a scale below 2^-100 may overflow: divide instead
  float r = rintf(s >= 7.9e-31f ? x * inv : __fdiv_rn(x, s));
  const float e = fmaf(-r, s, x);
  const float twice = fabsf(e) + fabsf(e);
  const bool odd = (static_cast<int>(r) & 1) != 0;
  if (twice > s || (twice == s && odd)) r += copysignf(1.0f, e);
  return static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
}

// An earlier code under a larger scale: c s / s' has at most 31 significant
// bits above and 24 below the line, so a quotient that is no tie is further
// from one than a double's rounding.
__device__ __forceinline__ int Requantise(int c, double from, double to) {
  return static_cast<int>(rint(static_cast<double>(c) * from / to));
}

struct Kv8WriteArgs {
  Kv8Rows at;
  int8_t* codes[2];
  float* scales[2];
  const float* x[2];
};

// CTA = (touched block, kv head, K or V).  The new rows pass through shared
// memory once (their maximum, then their codes).
__global__ void __launch_bounds__(kKv8Threads) Kv8WriteKernel(Kv8WriteArgs a) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  extern __shared__ __align__(16) float rows[];  // [count][hd]
  __shared__ uint32_t top_of[kKv8Threads / 32];
  const Kv8Span s = FindSpan(a.at, blockIdx.x);
  if (s.block < 0 || s.count == 0) return;
  const int which = blockIdx.z, head = blockIdx.y;
  const int hd = a.at.hd, B = a.at.block, hd4 = hd >> 2;
  const float* x = a.x[which] + (s.row * a.at.kv_heads + head) * hd;
  const int64_t row_stride = static_cast<int64_t>(a.at.kv_heads) * hd;
  // magnitudes as integers: NaN above Inf above every number
  uint32_t top = 0;
  for (int i = threadIdx.x; i < s.count * hd4; i += kKv8Threads) {
    const int t = i / hd4, c = i - t * hd4;
    const float4 v = LoadStream(reinterpret_cast<const float4*>(x + t * row_stride) + c);
    reinterpret_cast<float4*>(rows)[i] = v;
    top = max(max(top, __float_as_uint(v.x) & 0x7fffffffu),
              max(__float_as_uint(v.y) & 0x7fffffffu,
                  max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) top_of[threadIdx.x >> 5] = top;
  float* scale_at = a.scales[which] + s.block * a.at.kv_heads + head;
  const float had = s.first > 0 ? *scale_at : 0.0f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kKv8Threads / 32; ++w) top = max(top, top_of[w]);
  const float fresh = __fdiv_rn(__uint_as_float(top), 127.0f);
  const float scale =
      __float_as_uint(fresh) > (__float_as_uint(had) & 0x7fffffffu) ? fresh : had;
  if (threadIdx.x == 0) *scale_at = scale;  // every thread has read it
  const bool usable = scale > 0.0f && scale < INFINITY;
  const float inv = 1.0f / scale;
  const bool moved = scale != had;
  int8_t* codes = a.codes[which] + (s.block * a.at.kv_heads + head) * static_cast<int64_t>(B) * hd;
  const auto code = [&](int t, int d, int old) -> int {  // token t of the block, dimension d
    if (!usable) return 0;
    if (t < s.first) return moved ? Requantise(old, had, scale) : old;
    if (t >= s.first + s.count) return 0;
    return Quantise(rows[(t - s.first) * hd + d], scale, inv);
  };
  if (which == 0) {  // [B][hd]: 4 dimensions of a token
    for (int i = threadIdx.x; i < B * hd4; i += kKv8Threads) {
      const int t = i / hd4, d = 4 * (i - t * hd4);
      char4 c = t < s.first ? reinterpret_cast<char4*>(codes)[i] : make_char4(0, 0, 0, 0);
      c = make_char4(code(t, d, c.x), code(t, d + 1, c.y), code(t, d + 2, c.z),
                     code(t, d + 3, c.w));
      reinterpret_cast<char4*>(codes)[i] = c;
    }
  } else {  // [hd][B]: 16 tokens of a dimension, neighbouring lanes neighbouring dimensions
    for (int i = threadIdx.x; i < hd * (B >> 4); i += kKv8Threads) {
      const int d = i % hd, t0 = 16 * (i / hd);
      uint4* at = reinterpret_cast<uint4*>(codes + d * B + t0);
      uint32_t w[4] = {0, 0, 0, 0};
      if (t0 < s.first) {
        const uint4 old = *at;
        w[0] = old.x; w[1] = old.y; w[2] = old.z; w[3] = old.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t packed = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int old = static_cast<int8_t>(w[j] >> (8 * e));
          packed |= (static_cast<uint32_t>(code(t0 + 4 * j + e, d, old)) & 0xffu) << (8 * e);
        }
        w[j] = packed;
      }
      *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

struct Kv8ReadArgs {
  Kv8Rows at;
  const int8_t* codes[2];
  const float* scales[2];
  float* x[2];
};

// CTA = (touched block, kv head, K or V).
__global__ void __launch_bounds__(kKv8Threads) Kv8ReadKernel(Kv8ReadArgs a) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  const Kv8Span s = FindSpan(a.at, blockIdx.x);
  const int which = blockIdx.z, head = blockIdx.y;
  if (s.count == 0 || a.x[which] == nullptr) return;
  const int hd = a.at.hd, B = a.at.block, hd4 = hd >> 2;
  float* x = a.x[which] + (s.row * a.at.kv_heads + head) * hd;
  const int64_t row_stride = static_cast<int64_t>(a.at.kv_heads) * hd;
  if (s.block < 0) {
    for (int i = threadIdx.x; i < s.count * hd4; i += kKv8Threads)
      reinterpret_cast<float4*>(x + (i / hd4) * row_stride)[i % hd4] =
          make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  const float scale = a.scales[which][s.block * a.at.kv_heads + head];
  const int8_t* codes =
      a.codes[which] + (s.block * a.at.kv_heads + head) * static_cast<int64_t>(B) * hd;
  if (which == 0) {
    for (int i = threadIdx.x; i < s.count * hd4; i += kKv8Threads) {
      const int t = i / hd4, c = i - t * hd4;
      const char4 v = reinterpret_cast<const char4*>(codes + (s.first + t) * hd)[c];
      StoreStream(reinterpret_cast<float4*>(x + t * row_stride) + c,
                  make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale));
    }
  } else {
    for (int i = threadIdx.x; i < hd * (B >> 4); i += kKv8Threads) {
      const int d = i % hd, t0 = 16 * (i / hd);
      if (t0 + 16 <= s.first || t0 >= s.first + s.count) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(codes + d * B + t0);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int t = t0 + j - s.first;
        if (t >= 0 && t < s.count)
          x[t * row_stride + d] =
              static_cast<float>(static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3)))) * scale;
      }
    }
  }
}

// The shape rules that the cache's entries share; nullptr when they hold.
const char* Kv8Shape(int64_t n_blocks, int block_tokens, int64_t table_cols, int64_t n_seqs,
                     int kv_heads, int hd) {
  if (block_tokens != 32 && block_tokens != 64 && block_tokens != 128)
    return "block_tokens must be 32, 64 or 128";
  if (kv_heads <= 0 || kv_heads > 65535 || hd <= 0 || hd % 32 != 0 || hd > 256)
    return "kv heads in [1, 65535], head_dim % 32 == 0, head_dim <= 256";
  if (n_blocks < 0 || n_blocks > INT_MAX || table_cols < 0 || table_cols > INT_MAX / block_tokens ||
      n_seqs < 0 || n_seqs > INT_MAX / 8)
    return "bad n_blocks, table_cols or n_seqs";
  return nullptr;
}

// Blocks that `rows` rows of n_seqs sequences touch at most: a sequence of n
// rows touches at most n, and at most n / B + 2.
int64_t MostTouched(int64_t rows, int64_t n_seqs, int block) {
  const int64_t by_seq = rows / block + 2 * n_seqs;
  return rows < by_seq ? rows : by_seq;
}

int Kv8Check(const char* op, bool null, bool aligned, int64_t n_blocks, int block_tokens,
             int64_t table_cols, int64_t n_seqs, int64_t rows, int kv_heads, int hd) {
  const std::string name(op);
  if (const char* bad = Kv8Shape(n_blocks, block_tokens, table_cols, n_seqs, kv_heads, hd))
    return Fail(MLB_ERR_ARG, name + ": " + bad);
  if (rows < 0 || rows > INT_MAX / 8) return Fail(MLB_ERR_ARG, name + ": bad rows");
  if (rows == 0 || n_seqs == 0) return MLB_OK;
  if (null) return Fail(MLB_ERR_ARG, name + ": null pointer");
  if (!aligned) return Fail(MLB_ERR_ARG, name + ": codes, k and v must be 16-byte aligned");
  return MLB_OK;
}

// ---------------------------------------------------------------------------
// Eviction.

constexpr int kEvictThreads = 1024;

struct EvictArgs {
  const int32_t* table;
  const int32_t* lengths;
  const float* mass;
  int32_t* table_out;
  int32_t* lengths_out;
  float* mass_out;
  int32_t* freed;
  int64_t cols;
  int64_t keep, sink, recent;
  int block;
  int32_t* status;
};

// Order of the masses as unsigned integers: NaN largest, -0 as 0.
__device__ __forceinline__ uint32_t MassKey(float m) {
  if (m != m) return 0xffffffffu;
  const uint32_t b = __float_as_uint(m + 0.0f);
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

// CTA = one sequence.  The g-th smallest key of the candidates is found digit
// by digit (four 8-bit histograms); everything below it leaves, and of the
// keys equal to it the first ones that are still wanted.  A prefix count
// then closes up ids and masses.
__global__ void __launch_bounds__(kEvictThreads) EvictKernel(EvictArgs a) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  __shared__ int hist[256];
  __shared__ int digit_of, below_digit;
  __shared__ int warp_eq[kEvictThreads / 32], warp_leave[kEvictThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * a.cols;
  const int32_t length = a.lengths[blockIdx.x];
  int64_t blocks = (static_cast<int64_t>(length) + a.block - 1) / a.block;
  const bool bad = length < 0 || blocks > a.cols;
  if (bad) {
    if (threadIdx.x == 0) Raise(a.status, MLB_STATUS_BAD_LENGTH);
    blocks = a.cols;
  }
  const int64_t gone = bad || blocks <= a.keep ? 0 : blocks - a.keep;
  const int64_t lo = a.sink, hi = blocks - a.recent;  // candidates (when gone > 0)
  uint32_t threshold = 0;
  int64_t equal = 0;  // keys equal to the threshold that leave
  if (gone > 0) {
    int64_t want = gone;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int64_t i = lo + threadIdx.x; i < hi; i += kEvictThreads) {
        const uint32_t key = MassKey(a.mass[row + i]);
        if ((key & mask) == (threshold & mask)) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {  // the digit at which the count reaches want
        int each[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += each[j] = hist[8 * lane + j];
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        int before = upto - sum;
        if (before < want && want <= upto) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (before < want && want <= before + each[j]) {
              digit_of = 8 * lane + j;
              below_digit = before;
            }
            before += each[j];
          }
        }
      }
      __syncthreads();
      threshold |= static_cast<uint32_t>(digit_of) << shift;
      want -= below_digit;
    }
    equal = want;
  }
  // close up, kEvictThreads places at a time: a place is read before any
  // place at or before it is written, so outputs may be the inputs
  int64_t seen_eq = 0, left = 0;
  for (int64_t base = 0; base < blocks; base += kEvictThreads) {
    const int64_t i = base + threadIdx.x;
    const bool in = i < blocks;
    const int32_t id = in ? a.table[row + i] : -1;
    const float m = in ? a.mass[row + i] : 0.0f;
    const bool open = gone > 0 && i >= lo && i < hi;
    const uint32_t key = MassKey(m);
    const bool eq = open && key == threshold;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[warp] = __popc(eqs);
    __syncthreads();
    int64_t my_eq = seen_eq + __popc(eqs & ((1u << lane) - 1));
#pragma unroll 4
    for (int w = 0; w < kEvictThreads / 32; ++w) {
      if (w < warp) my_eq += warp_eq[w];
      seen_eq += warp_eq[w];
    }
    const bool leaves = open && (key < threshold || (eq && my_eq < equal));
    const uint32_t leave = __ballot_sync(0xffffffffu, leaves);
    if (lane == 0) warp_leave[warp] = __popc(leave);
    __syncthreads();
    int64_t my_left = left + __popc(leave & ((1u << lane) - 1));
#pragma unroll 4
    for (int w = 0; w < kEvictThreads / 32; ++w) {
      if (w < warp) my_left += warp_leave[w];
      left += warp_leave[w];
    }
    if (in && leaves && a.freed != nullptr) a.freed[row + my_left] = id;
    if (in && !leaves) {
      a.table_out[row + i - my_left] = id;
      a.mass_out[row + i - my_left] = m;
    }
    __syncthreads();  // the counters are read before they are filled again
  }
  if (!bad)
    for (int64_t i = blocks - left + threadIdx.x; i < a.cols; i += kEvictThreads) {
      a.table_out[row + i] = -1;
      a.mass_out[row + i] = 0.0f;
    }
  if (a.freed != nullptr)
    for (int64_t i = left + threadIdx.x; i < a.cols; i += kEvictThreads) a.freed[row + i] = -1;
  if (threadIdx.x == 0) a.lengths_out[blockIdx.x] = length - static_cast<int32_t>(left) * a.block;
}

}  // namespace
}  // namespace mlb

extern "C" int mlb_kv8_write_f32(int8_t* k_codes, int8_t* v_codes, float* k_scales,
                                 float* v_scales, int64_t n_blocks, int block_tokens,
                                 const int32_t* table, int64_t table_cols, int64_t n_seqs,
                                 const float* k, const float* v, const int32_t* offsets,
                                 const int32_t* positions, int64_t rows, int n_kv_heads,
                                 int head_dim, int32_t* status, void* stream) {
  using namespace mlb;
  const int rc = Kv8Check(
      "mlb_kv8_write_f32",
      k_codes == nullptr || v_codes == nullptr || k_scales == nullptr || v_scales == nullptr ||
          table == nullptr || k == nullptr || v == nullptr || offsets == nullptr ||
          positions == nullptr,
      Aligned16(k_codes) && Aligned16(v_codes) && Aligned16(k) && Aligned16(v), n_blocks,
      block_tokens, table_cols, n_seqs, rows, n_kv_heads, head_dim);
  if (rc != MLB_OK || rows == 0 || n_seqs == 0) return rc;
  Kv8WriteArgs a{};
  a.at = Kv8Rows{table, offsets, positions, table_cols, n_blocks, rows,
                 static_cast<int>(n_seqs), block_tokens, n_kv_heads, head_dim, status};
  a.codes[0] = k_codes;
  a.codes[1] = v_codes;
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.x[0] = k;
  a.x[1] = v;
  const int shm = block_tokens * head_dim * 4;
  if (shm > 48 * 1024 &&
      cudaFuncSetAttribute(Kv8WriteKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shm) !=
          cudaSuccess) {
    cudaGetLastError();
    return Fail(MLB_ERR_CUDA, "mlb_kv8_write_f32: shared memory opt-in");
  }
  const dim3 grid(static_cast<unsigned>(MostTouched(rows, n_seqs, block_tokens)),
                  static_cast<unsigned>(n_kv_heads), 2);
  Launch(Kv8WriteKernel, grid, kKv8Threads, static_cast<size_t>(shm), AsStream(stream), a);
  return CheckLaunch("mlb_kv8_write_f32");
}

extern "C" int mlb_kv8_read_f32(const int8_t* k_codes, const int8_t* v_codes,
                                const float* k_scales, const float* v_scales, int64_t n_blocks,
                                int block_tokens, const int32_t* table, int64_t table_cols,
                                int64_t n_seqs, float* k, float* v, const int32_t* offsets,
                                const int32_t* positions, int64_t rows, int n_kv_heads,
                                int head_dim, int32_t* status, void* stream) {
  using namespace mlb;
  const int rc = Kv8Check(
      "mlb_kv8_read_f32",
      k_codes == nullptr || v_codes == nullptr || k_scales == nullptr || v_scales == nullptr ||
          table == nullptr || (k == nullptr && v == nullptr) || offsets == nullptr ||
          positions == nullptr,
      Aligned16(k_codes) && Aligned16(v_codes) && Aligned16(k) && Aligned16(v), n_blocks,
      block_tokens, table_cols, n_seqs, rows, n_kv_heads, head_dim);
  if (rc != MLB_OK || rows == 0 || n_seqs == 0) return rc;
  Kv8ReadArgs a{};
  a.at = Kv8Rows{table, offsets, positions, table_cols, n_blocks, rows,
                 static_cast<int>(n_seqs), block_tokens, n_kv_heads, head_dim, status};
  a.codes[0] = k_codes;
  a.codes[1] = v_codes;
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.x[0] = k;
  a.x[1] = v;
  const dim3 grid(static_cast<unsigned>(MostTouched(rows, n_seqs, block_tokens)),
                  static_cast<unsigned>(n_kv_heads), 2);
  Launch(Kv8ReadKernel, grid, kKv8Threads, 0, AsStream(stream), a);
  return CheckLaunch("mlb_kv8_read_f32");
}

extern "C" int mlb_kv8_evict(const int32_t* table, int64_t table_cols, const int32_t* lengths,
                             const float* mass, int64_t n_seqs, int block_tokens,
                             int64_t keep_blocks, int64_t sink_blocks, int64_t recent_blocks,
                             int32_t* table_out, int32_t* lengths_out, float* mass_out,
                             int32_t* freed, int32_t* status, void* stream) {
  using namespace mlb;
  if (const char* bad = Kv8Shape(0, block_tokens, table_cols, n_seqs, 1, 32))
    return Fail(MLB_ERR_ARG, std::string("mlb_kv8_evict: ") + bad);
  if (sink_blocks < 0 || recent_blocks < 1 || sink_blocks > INT_MAX || recent_blocks > INT_MAX ||
      sink_blocks + recent_blocks > keep_blocks)
    return Fail(MLB_ERR_ARG,
                "mlb_kv8_evict: sink >= 0, recent >= 1 and sink + recent <= keep blocks");
  if (n_seqs == 0) return MLB_OK;
  if (lengths == nullptr || lengths_out == nullptr ||
      (table_cols > 0 && (table == nullptr || mass == nullptr || table_out == nullptr ||
                          mass_out == nullptr)))
    return Fail(MLB_ERR_ARG, "mlb_kv8_evict: null pointer");
  const EvictArgs a{table, lengths,    mass,        table_out,   lengths_out,   mass_out, freed,
                    table_cols, keep_blocks, sink_blocks, recent_blocks, block_tokens, status};
  Launch(EvictKernel, static_cast<unsigned>(n_seqs), kEvictThreads, 0, AsStream(stream), a);
  return CheckLaunch("mlb_kv8_evict");
}
