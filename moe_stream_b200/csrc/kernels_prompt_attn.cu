// kernels_prompt_attn.cu — causal attention of packed sequences of different lengths (grouped heads, sliding
// window, sinks, keys of a cached prefix in front of the queries).
#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kWarps = 4;

// one warp per (query, head): lanes hold the dims, keys in order with a running maximum and sum
template <class T, int HD>
__global__ void __launch_bounds__(kWarps * 32) prompt_attn_kernel(const ms_prompt_attn a, uint32_t* err) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31, h = blockIdx.y, g = h / (a.heads / a.kv_heads);
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.total_q) return;
  const int seq = seq_of_row(a.cu_q, a.n_seqs, row);
  if (seq < 0) return;
  const int k0 = a.cu_k[seq], k1 = a.cu_k[seq + 1];
  if (k0 < 0 || k1 < k0 || k1 > a.total_k) {
    if (lane == 0) atomicOr(err, EF_BAD_INDEX);
    return;
  }
  const int last = k1 - (a.cu_q[seq + 1] - row), first = a.window > 0 ? max(k0, last - a.window + 1) : k0;
  float qv[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) { qv[i] = to_f32(((const T*)a.q)[row * a.q_stride + h * HD + lane + 32 * i]); o[i] = 0.f; }
  for (int j = first; j <= last; ++j) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(qv[i], to_f32(((const T*)a.k)[j * a.k_stride + g * HD + lane + 32 * i]), s);
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + p * to_f32(((const T*)a.v)[j * a.v_stride + g * HD + lane + 32 * i]);
    m = mn;
  }
  if (a.sinks) {
    const float mn = fmaxf(m, a.sinks[h]), f = expf(m - mn);
    l = l * f + expf(a.sinks[h] - mn);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    ((T*)a.out)[row * a.out_stride + h * HD + lane + 32 * i] = from_f32<T>(l > 0.f ? o[i] / l : 0.f);
}

template <class T>
cudaError_t start(const DevCtx& d, const ms_prompt_attn& a, cudaStream_t s) {
  const dim3 grid((a.total_q + kWarps - 1) / kWarps, a.heads);
  if (a.head_dim == 64) prompt_attn_kernel<T, 64><<<grid, kWarps * 32, 0, s>>>(a, d.err);
  else if (a.head_dim == 128) prompt_attn_kernel<T, 128><<<grid, kWarps * 32, 0, s>>>(a, d.err);
  else prompt_attn_kernel<T, 256><<<grid, kWarps * 32, 0, s>>>(a, d.err);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prompt_attention(const DevCtx& d, const ms_prompt_attn& a, cudaStream_t s) {
  if (a.total_q == 0 || a.n_seqs == 0) return cudaSuccess;
  return a.type == MS_Q_F16 ? start<__half>(d, a, s) : start<__nv_bfloat16>(d, a, s);
}

}  // namespace ms
