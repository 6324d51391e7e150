// kernels_kv4_attn.cu — attention of the newest tokens of each sequence over the paged 4-bit K/V cache.
#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace ms {
namespace {

constexpr int kWarps = 4;

template <int HD>
__device__ __forceinline__ float k_value(const uint8_t* blk, int tok, int dim) {
  constexpr int G = HD / 32;
  const int w = dim >> 5, t = (dim >> 3) & 3, n = (dim >> 1) & 3, h = dim & 1;
  const uint32_t word = reinterpret_cast<const uint32_t*>(blk)[tok * 4 * G + t * G + w];
  const float2 s = unpack2<__half>(reinterpret_cast<const uint32_t*>(blk + kv4_k_scales(HD))[tok * G + w]);
  return fmaf(s.x, (float)(16 + ((word >> (4 * n + 16 * h)) & 15u)), s.y);
}
template <int HD>
__device__ __forceinline__ float v_value(const uint8_t* blk, int tok, int dim) {
  constexpr int G = HD / 32;
  const int pair = tok >> 1, par = tok & 1, C = dim >> 4;
  const uint16_t q = reinterpret_cast<const uint16_t*>(
      blk + kv4_v_codes(HD))[(pair * (HD / 16) + kv4_v_chunk<HD>(C, pair)) * 8 + ((dim >> 2) & 3) * 2 + par];
  const uint16_t* s = reinterpret_cast<const uint16_t*>(blk + kv4_v_scales(HD)) + (pair * G + (dim >> 5)) * 4 + par;
  return fmaf(h2f_bits(s[0]), (float)(16 + ((q >> (4 * (dim & 3))) & 15u)), h2f_bits(s[2]));
}

// one block per (query row, sequence): warps take every fourth key, lanes the dims; the warps' running maxima,
// sums and outputs are joined at the end
template <class T, int HD>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_kernel(const ms_kv4_cache c, const ms_kv4_attn a, uint32_t* err) {
  constexpr int N = HD / 32;
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seq = blockIdx.y;
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads, g = h / (a.heads / c.kv_heads);
  int len = a.lens[seq];
  if (len < 0 || len > c.max_pages * c.page_tokens) {
    if (threadIdx.x == 0) atomicOr(err, EF_BAD_INDEX);
    len = len < 0 ? 0 : c.max_pages * c.page_tokens;
  }
  const int last = len - a.n_query + t, first = a.window > 0 ? max(0, last - a.window + 1) : 0;
  const int64_t row = ((int64_t)seq * a.n_query + t) * a.heads + h;
  const T* q = (const T*)a.q + row * HD;
  float qv[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) { qv[i] = to_f32(q[lane + 32 * i]); o[i] = 0.f; }
  for (int j = first + warp; j <= last; j += kWarps) {
    const uint8_t* blk = kv4_block(c, seq, j, g);
    if (!blk) {
      if (lane == 0) atomicOr(err, EF_BAD_INDEX);
      continue;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(qv[i], k_value<HD>(blk, j & 15, lane + 32 * i), s);
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + p * v_value<HD>(blk, j & 15, lane + 32 * i);
    m = mn;
  }
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
  for (int i = 0; i < N; ++i) sm_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  if (warp) return;
  float mm = a.sinks ? a.sinks[h] : -INFINITY;
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w]);
  float ll = a.sinks ? expf(a.sinks[h] - mm) : 0.f, r[N] = {};
  for (int w = 0; w < kWarps; ++w) {
    if (sm_m[w] == -INFINITY) continue;
    const float f = expf(sm_m[w] - mm);
    ll += sm_l[w] * f;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] += sm_o[w][lane + 32 * i] * f;
  }
  T* out = (T*)a.out + row * HD;
#pragma unroll
  for (int i = 0; i < N; ++i) out[lane + 32 * i] = from_f32<T>(ll > 0.f ? r[i] / ll : 0.f);
}

template <class T>
cudaError_t start(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_attn& a, cudaStream_t s) {
  const dim3 grid(a.n_query * a.heads, c.n_seqs);
  if (c.head_dim == 64) kv4_attn_kernel<T, 64><<<grid, kWarps * 32, 0, s>>>(c, a, d.err);
  else if (c.head_dim == 128) kv4_attn_kernel<T, 128><<<grid, kWarps * 32, 0, s>>>(c, a, d.err);
  else kv4_attn_kernel<T, 256><<<grid, kWarps * 32, 0, s>>>(c, a, d.err);
  return cudaGetLastError();
}

}  // namespace

size_t kv4_attn_workspace(const DevCtx&, const ms_kv4_cache&, int, int) { return 16; }

cudaError_t launch_kv4_attention(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_attn& a, cudaStream_t s) {
  if (c.n_seqs == 0) return cudaSuccess;
  return a.type == MS_Q_F16 ? start<__half>(d, c, a, s) : start<__nv_bfloat16>(d, c, a, s);
}

}  // namespace ms
