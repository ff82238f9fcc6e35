// Causal attention over packed sequences.
//
// Sequence i has Q query rows and K keys; its row r sees keys
// 0 .. K - Q + r:  out = softmax(q k^T / sqrt(hd)) v, kv head h / G for query
// head h.  Rows and keys of a sequence are found from the offsets on the
// device.
#include <climits>
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace mlb {
namespace {

constexpr int kPkWarps = 4;
constexpr int kPkMaxGroup = 8;

struct PkArgs {
  const float* q;
  const float* k;
  const float* v;
  float* out;
  const int32_t* q_offsets;
  const int32_t* k_offsets;
  int64_t q_rows;
  int64_t k_rows;
  int n_seqs;
  int n_heads;
  int kv_heads;
  int hd;
  float scale;
  int32_t* status;
};

struct PkSeq {
  int64_t q0, q1, k0, k1;
};

// Sequence i's ranges; false (and the status bit, once per launch) when they
// are not inside the tensors.
__device__ __forceinline__ bool PkRange(const PkArgs& a, int i, PkSeq& s) {
  s.q0 = a.q_offsets[i];
  s.q1 = a.q_offsets[i + 1];
  s.k0 = a.k_offsets[i];
  s.k1 = a.k_offsets[i + 1];
  return s.q0 >= 0 && s.q1 >= s.q0 && s.q1 <= a.q_rows && s.k0 >= 0 && s.k1 >= s.k0 &&
         s.k1 <= a.k_rows;
}

// Any head size up to 256 and any alignment of the sequences: CTA = (query
// row, kv head), 4 warps share the row's keys, each with an online softmax
// for the G heads of the group; the warps' states are merged at the end.
template <int G, int NV>
__global__ void __launch_bounds__(kPkWarps * 32) PkRowKernel(PkArgs a) {
  LaunchWait();  // the previous kernel on the stream has completed
  LaunchNext();
  __shared__ float sm_m[kPkWarps][G];
  __shared__ float sm_l[kPkWarps][G];
  __shared__ float4 sm_acc[kPkWarps][G][32 * NV];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int g = blockIdx.y, hd4 = a.hd >> 2;
  // the sequence that holds the row: its ranges, or none
  PkSeq s{};
  bool have = false;
  for (int base = 0; base < a.n_seqs; base += 32) {
    const int i = base + lane;
    PkSeq mine{};
    bool in = false;
    if (i < a.n_seqs) {
      const bool good = PkRange(a, i, mine);
      if (!good && row == 0 && g == 0 && warp == 0 && a.status != nullptr)
        atomicOr(a.status, MLB_STATUS_BAD_LENGTH);
      in = good && row >= mine.q0 && row < mine.q1;
    }
    const uint32_t found = __ballot_sync(0xffffffffu, in);
    if (found != 0 && !have) {
      const int src = __ffs(found) - 1;
      s.q0 = __shfl_sync(0xffffffffu, mine.q0, src);
      s.q1 = __shfl_sync(0xffffffffu, mine.q1, src);
      s.k0 = __shfl_sync(0xffffffffu, mine.k0, src);
      s.k1 = __shfl_sync(0xffffffffu, mine.k1, src);
      have = true;
    }
    if (have && row != 0) break;  // row 0 looks at every sequence's ranges
  }
  if (!have) return;
  const int64_t visible = (s.k1 - s.k0) - (s.q1 - row) + 1;  // keys the row sees
  const int64_t q_at = (row * a.n_heads + static_cast<int64_t>(g) * G) * hd4;
  const float4* q4 = reinterpret_cast<const float4*>(a.q) + q_at;
  float4 q[G][NV];
  float m[G], l[G];
  float4 acc[G][NV];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = lane + 32 * v;
      q[h][v] = i < hd4 ? q4[h * hd4 + i] : make_float4(0.f, 0.f, 0.f, 0.f);
      acc[h][v] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  const int64_t stride4 = static_cast<int64_t>(a.kv_heads) * hd4;
  const float4* k4 = reinterpret_cast<const float4*>(a.k) + s.k0 * stride4 + g * hd4;
  const float4* v4 = reinterpret_cast<const float4*>(a.v) + s.k0 * stride4 + g * hd4;
  for (int64_t t = warp; t < visible; t += kPkWarps) {
    float4 kk[NV], vv[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = lane + 32 * v;
      kk[v] = i < hd4 ? k4[t * stride4 + i] : make_float4(0.f, 0.f, 0.f, 0.f);
      vv[v] = i < hd4 ? v4[t * stride4 + i] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float dot = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        dot = fmaf(q[h][v].x, kk[v].x, dot);
        dot = fmaf(q[h][v].y, kk[v].y, dot);
        dot = fmaf(q[h][v].z, kk[v].z, dot);
        dot = fmaf(q[h][v].w, kk[v].w, dot);
      }
      const float score = WarpSum(dot) * a.scale;
      const float m_new = fmaxf(m[h], score);
      const float alpha = m[h] == -INFINITY ? 0.0f : expf(m[h] - m_new);
      const float p = expf(score - m_new);
      l[h] = fmaf(l[h], alpha, p);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        acc[h][v].x = fmaf(acc[h][v].x, alpha, p * vv[v].x);
        acc[h][v].y = fmaf(acc[h][v].y, alpha, p * vv[v].y);
        acc[h][v].z = fmaf(acc[h][v].z, alpha, p * vv[v].z);
        acc[h][v].w = fmaf(acc[h][v].w, alpha, p * vv[v].w);
      }
      m[h] = m_new;
    }
  }
#pragma unroll
  for (int h = 0; h < G; ++h) {
    if (lane == 0) {
      sm_m[warp][h] = m[h];
      sm_l[warp][h] = l[h];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) sm_acc[warp][h][lane + 32 * v] = acc[h][v];
  }
  __syncthreads();
  for (int h = warp; h < G; h += kPkWarps) {
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < kPkWarps; ++w) mm = fmaxf(mm, sm_m[w][h]);
    float f[kPkWarps];
#pragma unroll
    for (int w = 0; w < kPkWarps; ++w) {
      f[w] = sm_m[w][h] == -INFINITY ? 0.0f : expf(sm_m[w][h] - mm);
      // a warp whose scores are NaN keeps them visible
      if (sm_l[w][h] != sm_l[w][h]) f[w] = NAN;
      ll = fmaf(sm_l[w][h], f[w], ll);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = lane + 32 * v;
      if (i >= hd4) continue;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPkWarps; ++w) {
        const float4 x = sm_acc[w][h][i];
        o.x = fmaf(x.x, f[w], o.x);
        o.y = fmaf(x.y, f[w], o.y);
        o.z = fmaf(x.z, f[w], o.z);
        o.w = fmaf(x.w, f[w], o.w);
      }
      if (visible > 0) o = make_float4(o.x / ll, o.y / ll, o.z / ll, o.w / ll);
      reinterpret_cast<float4*>(a.out)[q_at + h * hd4 + i] = o;
    }
  }
}

template <int G>
void LaunchPkRows(const PkArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.q_rows), static_cast<unsigned>(a.kv_heads));
  if (a.hd <= 128)
    Launch(PkRowKernel<G, 1>, grid, kPkWarps * 32, 0, s, a);
  else
    Launch(PkRowKernel<G, 2>, grid, kPkWarps * 32, 0, s, a);
}

const char* PkShape(int64_t q_rows, int64_t k_rows, int64_t n_seqs, int n_heads, int kv_heads,
                    int hd) {
  if (n_heads <= 0 || kv_heads <= 0 || n_heads % kv_heads != 0 ||
      n_heads / kv_heads > kPkMaxGroup || kv_heads > 65535 || hd <= 0 || hd % 4 != 0 || hd > 256)
    return "heads must divide, group <= 8, head_dim % 4 == 0, head_dim <= 256";
  if (q_rows < 0 || k_rows < 0 || n_seqs < 0 || q_rows > INT_MAX / 8 || k_rows > INT_MAX / 8 ||
      n_seqs > INT_MAX / 8)
    return "bad q_rows, k_rows or n_seqs";
  return nullptr;
}

}  // namespace
}  // namespace mlb

extern "C" int64_t mlb_attention_packed_scratch_floats(int64_t q_rows, int64_t k_rows,
                                                       int64_t n_seqs, int n_heads,
                                                       int n_kv_heads, int head_dim) {
  using namespace mlb;
  if (PkShape(q_rows, k_rows, n_seqs, n_heads, n_kv_heads, head_dim) != nullptr) return -1;
  return 0;
}

extern "C" int mlb_attention_packed_f32(const float* q, const float* k, const float* v, float* out,
                                        const int32_t* q_offsets, const int32_t* k_offsets,
                                        int64_t n_seqs, int64_t q_rows, int64_t k_rows,
                                        int n_heads, int n_kv_heads, int head_dim, float* scratch,
                                        int64_t scratch_floats, int32_t* status, void* stream) {
  using namespace mlb;
  const std::string op("mlb_attention_packed_f32: ");
  if (const char* bad = PkShape(q_rows, k_rows, n_seqs, n_heads, n_kv_heads, head_dim))
    return Fail(MLB_ERR_ARG, op + bad);
  if (q_rows == 0 || n_seqs == 0) return MLB_OK;
  if (q == nullptr || out == nullptr || q_offsets == nullptr || k_offsets == nullptr ||
      (k_rows > 0 && (k == nullptr || v == nullptr)))
    return Fail(MLB_ERR_ARG, op + "null pointer");
  if (!Aligned16(q) || !Aligned16(k) || !Aligned16(v) || !Aligned16(out) || !Aligned16(scratch))
    return Fail(MLB_ERR_ARG, op + "q, k, v, out and scratch must be 16-byte aligned");
  const int64_t need = mlb_attention_packed_scratch_floats(q_rows, k_rows, n_seqs, n_heads,
                                                           n_kv_heads, head_dim);
  if (need > 0 && (scratch == nullptr || scratch_floats < need))
    return Fail(MLB_ERR_ARG, op + "scratch too small");
  const PkArgs a{q, k, v, out, q_offsets, k_offsets, q_rows, k_rows, static_cast<int>(n_seqs),
                 n_heads, n_kv_heads, head_dim, 1.0f / std::sqrt(static_cast<float>(head_dim)),
                 status};
  cudaStream_t s = AsStream(stream);
  switch (n_heads / n_kv_heads) {
    case 1: LaunchPkRows<1>(a, s); break;
    case 2: LaunchPkRows<2>(a, s); break;
    case 3: LaunchPkRows<3>(a, s); break;
    case 4: LaunchPkRows<4>(a, s); break;
    case 5: LaunchPkRows<5>(a, s); break;
    case 6: LaunchPkRows<6>(a, s); break;
    case 7: LaunchPkRows<7>(a, s); break;
    default: LaunchPkRows<8>(a, s); break;
  }
  return CheckLaunch("mlb_attention_packed_f32");
}
