// Decode attention of several sequences over the 8-bit KV cache.
//
//   out[i][h] = softmax_t(q[i][h] . k_t / sqrt(hd)) . v_t,  t < lengths[i]
// with k_t, v_t = code * scale of the token's block (mlb_ops.h).  A unit is
// 32 consecutive tokens; it lies in one block, so it has one scale for K and
// one for V.  Online softmax over units; the weight that a block collects is
// found afterwards from each unit's (sum p, reference max) and the heads'
// final (M, L).
#include <climits>
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace mlb {
namespace {

constexpr int kUnit = 32;  // tokens
constexpr int kA8Threads = 128;
constexpr int kA8MaxGroup = 8;

struct A8Args {
  const float* q;
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scales;
  const float* v_scales;
  const int32_t* table;
  const int32_t* lengths;
  float* out;
  float2* lse;    // [n_seqs][n_heads] (M, L); L = 0: no token or a bad sequence
  float2* units;  // [n_seqs][unit columns][n_heads] (reference max, sum p), or null
  int64_t n_blocks;
  int64_t table_cols;
  int n_seqs;
  int block;
  int n_heads;
  int kv_heads;
  int hd;
  float scale;
  int32_t* status;
};

// CTA = (kv head, sequence): unit by unit, scores by (head, token) thread,
// weighted values by dimension thread.
__global__ void __launch_bounds__(kA8Threads) A8Kernel(A8Args a) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  __shared__ float qs[kA8MaxGroup * 256];
  __shared__ float p[kA8MaxGroup][kUnit];
  __shared__ float m_of[kA8MaxGroup], l_of[kA8MaxGroup], alpha_of[kA8MaxGroup];
  const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const int group = a.n_heads / a.kv_heads, hd = a.hd;
  const int64_t length = a.lengths[seq];
  const int32_t* table = a.table + seq * a.table_cols;
  bool bad = length < 0 || length > a.table_cols * a.block;
  if (bad && tid == 0 && a.status != nullptr) atomicOr(a.status, MLB_STATUS_BAD_LENGTH);
  const int64_t units = bad ? 0 : (length + kUnit - 1) / kUnit;
  const int64_t q0 = (static_cast<int64_t>(seq) * a.n_heads + head * group) * hd;
  for (int i = tid; i < group * hd; i += kA8Threads) qs[i] = a.q[q0 + i];
  if (tid < group) {
    m_of[tid] = -INFINITY;
    l_of[tid] = 0.0f;
  }
  float acc[kA8MaxGroup][2] = {};
  __syncthreads();
  for (int64_t u = 0; u < units; ++u) {
    const int64_t t0 = u * kUnit;
    const int n = static_cast<int>(length - t0 < kUnit ? length - t0 : kUnit);
    const int32_t id = table[t0 / a.block];
    if (id < 0 || id >= a.n_blocks) {
      bad = true;
      if (tid == 0 && a.status != nullptr) atomicOr(a.status, MLB_STATUS_BAD_BLOCK);
      break;  // the same for every thread
    }
    const int64_t at = static_cast<int64_t>(id) * a.kv_heads + head;
    const int place = static_cast<int>(t0 % a.block);
    const int8_t* k = a.k_codes + (at * a.block + place) * hd;
    const int8_t* v = a.v_codes + at * a.block * hd + place;
    const float ks = a.k_scales[at] * a.scale, vs = a.v_scales[at];
    for (int i = tid; i < group * kUnit; i += kA8Threads) {
      const int g = i / kUnit, t = i % kUnit;
      float dot = 0.0f;
      for (int d = 0; d < hd; ++d) dot = fmaf(qs[g * hd + d], static_cast<float>(k[t * hd + d]), dot);
      p[g][t] = t < n ? dot * ks : -INFINITY;
    }
    __syncthreads();
    for (int g = tid >> 5; g < group; g += kA8Threads / 32) {
      const int lane = tid & 31;
      const float s = p[g][lane];
      const float m_new = fmaxf(m_of[g], WarpMax(s));
      const float e = lane < n ? expf(s - m_new) : 0.0f;
      const float sum = WarpSum(e);
      p[g][lane] = e;
      if (lane == 0) {
        alpha_of[g] = expf(m_of[g] - m_new);
        l_of[g] = fmaf(l_of[g], alpha_of[g], sum);
        m_of[g] = m_new;
        if (a.units != nullptr)
          a.units[(seq * (a.table_cols * a.block / kUnit) + u) * a.n_heads + head * group + g] =
              make_float2(m_new, sum);
      }
    }
    __syncthreads();
    for (int j = 0; j < 2; ++j) {
      const int d = tid + j * kA8Threads;
      if (d >= hd) break;
      for (int g = 0; g < group; ++g) {
        float sum = 0.0f;
        for (int t = 0; t < n; ++t)
          sum = fmaf(p[g][t], static_cast<float>(v[static_cast<int64_t>(d) * a.block + t]), sum);
        acc[g][j] = fmaf(acc[g][j], alpha_of[g], sum * vs);
      }
    }
    __syncthreads();
  }
  const bool none = bad || units == 0;
  if (tid < group)
    a.lse[static_cast<int64_t>(seq) * a.n_heads + head * group + tid] =
        none ? make_float2(0.0f, 0.0f) : make_float2(m_of[tid], l_of[tid]);
  for (int j = 0; j < 2; ++j) {
    const int d = tid + j * kA8Threads;
    if (d >= hd) break;
    for (int g = 0; g < group; ++g) a.out[q0 + g * hd + d] = none ? 0.0f : acc[g][j] / l_of[g];
  }
}

// mass_out[i][c] = mass_in[i][c] + sum over heads and the block's units of
// (sum p) e^(m - M) / L.  A warp takes a column, its lanes the heads: the
// order of the sum is fixed.
__global__ void __launch_bounds__(256) A8MassKernel(A8Args a, const float* mass_in,
                                                    float* mass_out) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  const int lane = threadIdx.x & 31;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t seq = blockIdx.y;
  if (c >= a.table_cols) return;
  const int64_t length = a.lengths[seq];
  const int64_t unit_cols = a.table_cols * a.block / kUnit;
  const int64_t units = (length + kUnit - 1) / kUnit;
  const float2* lse = a.lse + seq * a.n_heads;
  float sum = 0.0f;
  if (length > 0 && length <= a.table_cols * a.block) {
    const int64_t u0 = c * (a.block / kUnit);
    const int64_t u1 = min(u0 + a.block / kUnit, units);
    for (int64_t u = u0; u < u1; ++u)
      for (int h = lane; h < a.n_heads; h += 32) {
        const float2 total = lse[h];  // L = 0: a bad block, nothing was collected
        const float2 x = a.units[(seq * unit_cols + u) * a.n_heads + h];
        if (total.y != 0.0f) sum += x.y * expf(x.x - total.x) / total.y;
      }
  }
  sum = WarpSum(sum);
  if (lane == 0) {
    const int64_t i = seq * a.table_cols + c;
    mass_out[i] = (mass_in != nullptr ? mass_in[i] : 0.0f) + sum;
  }
}

const char* A8Shape(int64_t n_seqs, int64_t table_cols, int block, int n_heads, int kv_heads,
                    int hd) {
  if (block != 32 && block != 64 && block != 128) return "block_tokens must be 32, 64 or 128";
  if (n_heads <= 0 || kv_heads <= 0 || n_heads % kv_heads != 0 ||
      n_heads / kv_heads > kA8MaxGroup || kv_heads > 65535 || hd <= 0 || hd % 32 != 0 || hd > 256)
    return "heads must divide, group <= 8, head_dim % 32 == 0, head_dim <= 256";
  if (n_seqs < 0 || n_seqs > 65535 || table_cols < 0 || table_cols > INT_MAX / block)
    return "bad n_seqs or table_cols";
  return nullptr;
}

struct A8Scratch {
  int64_t lse, units, total;  // floats: offsets and the sum
};

A8Scratch ScratchOf(int64_t n_seqs, int64_t table_cols, int block, int n_heads, bool with_mass) {
  A8Scratch s;
  s.lse = 0;
  s.units = (2 * n_seqs * n_heads + 3) & ~int64_t{3};
  s.total = s.units + (with_mass ? 2 * n_seqs * (table_cols * block / kUnit) * n_heads : 0);
  return s;
}

}  // namespace
}  // namespace mlb

extern "C" int64_t mlb_attention_kv8_scratch_floats(int64_t n_seqs, int64_t table_cols,
                                                    int block_tokens, int n_heads, int n_kv_heads,
                                                    int head_dim, int with_mass) {
  using namespace mlb;
  if (A8Shape(n_seqs, table_cols, block_tokens, n_heads, n_kv_heads, head_dim) != nullptr)
    return -1;
  return ScratchOf(n_seqs, table_cols, block_tokens, n_heads, with_mass != 0).total;
}

extern "C" int mlb_attention_kv8_f32(const float* q, const int8_t* k_codes, const int8_t* v_codes,
                                     const float* k_scales, const float* v_scales,
                                     int64_t n_blocks, int block_tokens, const int32_t* table,
                                     int64_t table_cols, const int32_t* lengths, int64_t n_seqs,
                                     int n_heads, int n_kv_heads, int head_dim, float* out,
                                     const float* mass_in, float* mass_out, float* scratch,
                                     int64_t scratch_floats, int32_t* status, void* stream) {
  using namespace mlb;
  const std::string op("mlb_attention_kv8_f32: ");
  if (const char* bad =
          A8Shape(n_seqs, table_cols, block_tokens, n_heads, n_kv_heads, head_dim))
    return Fail(MLB_ERR_ARG, op + bad);
  if (n_blocks < 0 || n_blocks > INT_MAX) return Fail(MLB_ERR_ARG, op + "bad n_blocks");
  if (n_seqs == 0) return MLB_OK;
  if (q == nullptr || out == nullptr || lengths == nullptr ||
      (table_cols > 0 && table == nullptr) ||
      (n_blocks > 0 && (k_codes == nullptr || v_codes == nullptr || k_scales == nullptr ||
                        v_scales == nullptr)))
    return Fail(MLB_ERR_ARG, op + "null pointer");
  if (mass_in != nullptr && mass_out == nullptr)
    return Fail(MLB_ERR_ARG, op + "mass_in without mass_out");
  if (!Aligned16(q) || !Aligned16(out) || !Aligned16(k_codes) || !Aligned16(v_codes) ||
      !Aligned16(scratch))
    return Fail(MLB_ERR_ARG, op + "q, out, codes and scratch must be 16-byte aligned");
  const A8Scratch need = ScratchOf(n_seqs, table_cols, block_tokens, n_heads, mass_out != nullptr);
  if (scratch == nullptr || scratch_floats < need.total)
    return Fail(MLB_ERR_ARG, op + "scratch too small");
  A8Args a{q, k_codes, v_codes, k_scales, v_scales, table, lengths, out,
           reinterpret_cast<float2*>(scratch + need.lse),
           mass_out != nullptr ? reinterpret_cast<float2*>(scratch + need.units) : nullptr,
           n_blocks, table_cols, static_cast<int>(n_seqs), block_tokens, n_heads, n_kv_heads,
           head_dim, 1.0f / std::sqrt(static_cast<float>(head_dim)), status};
  cudaStream_t s = AsStream(stream);
  Launch(A8Kernel, dim3(static_cast<unsigned>(n_kv_heads), static_cast<unsigned>(n_seqs)),
         kA8Threads, 0, s, a);
  if (mass_out != nullptr && table_cols > 0)
    Launch(A8MassKernel, dim3(static_cast<unsigned>((table_cols + 7) / 8),
                              static_cast<unsigned>(n_seqs)),
           256, 0, s, a, mass_in, mass_out);
  return CheckLaunch("mlb_attention_kv8_f32");
}
