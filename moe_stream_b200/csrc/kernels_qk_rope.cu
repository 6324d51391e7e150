// kernels_qk_rope.cu — per-head RMSNorm of queries and keys and the position rotation, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w   (per head; skipped without weights)
//   (a, b) -> (a cos - b sin, b cos + a sin)   on the first rot_dim dims, pairs (i, i + rot_dim / 2) or
//                                              (2 i, 2 i + 1), row pos[t] of the tables
//
// Everything is computed in f32 and rounded once to the output's type.  Bound by memory: each row is read and
// written once.  16,384 tokens of 16 + 2 heads of 256 dims (302 MB) take 58 us, 5.2 TB/s; a token's 36 heads of 128
// dims 1.6 us, a launch.
#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kThreads = 128;

// One group of LPR = head_dim / 16 lanes holds a head: two chunks of 8 dims per lane.  The first rot / 16 lanes hold
// the dims that rotate, 8 l .. and rot / 2 + 8 l .. (the two sides of their pairs, or 4 pairs of neighbours in each),
// the others share the rest the same way, so that the lanes of a load read neighbouring chunks.  A group takes
// HPG heads of one token, whose table row and norm weights stay in registers.
template <class TI, class TO, int LPR, int HPG, bool INTER>
__global__ void __launch_bounds__(kThreads, 5) qk_rope_kernel(const ms_qk_rope a, uint32_t* err) {
  const int lane = threadIdx.x % LPR;
  const uint32_t item = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const uint32_t nbq = (a.heads + HPG - 1) / HPG, nb = nbq + (a.kv_heads + HPG - 1) / HPG;
  const uint32_t t = item / nb, hb = item % nb;
  const bool is_q = hb < nbq;
  const int h0 = (is_q ? hb : hb - nbq) * HPG, nh = is_q ? a.heads : a.kv_heads;
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool in = t < (uint32_t)a.n_tokens;
  const int pos = in ? a.pos[t] : 0;
  // (loads that did not wait for the position took 65 us for 57 on a prompt of 16,384 tokens)
  const bool live = in && pos >= 0 && pos < a.max_pos;
  if (in && !live && hb == 0 && lane == 0) atomicOr(err, EF_BAD_INDEX);
  constexpr int HD = LPR * 16;
  const unsigned mask = (LPR == 32 ? 0xffffffffu : (1u << LPR) - 1) << (threadIdx.x % 32 / LPR * LPR);   // the lanes of the head
  const int half = a.rot_dim / 2, nt = a.rot_dim / 16;
  const bool turns = lane < nt;
  const int d0 = turns ? 8 * lane : a.rot_dim + 8 * (lane - nt), d1 = d0 + (turns ? half : 8 * (LPR - nt));
  const TI* src = (const TI*)(is_q ? a.q : a.k) + (int64_t)t * (is_q ? a.q_stride : a.k_stride);
  TO* dst = (TO*)(is_q ? a.q_out : a.k_out) + (int64_t)t * (is_q ? a.q_out_stride : a.k_out_stride);
  Raw8<TI> r[HPG][2];
#pragma unroll
  for (int i = 0; i < HPG; ++i)
    if (live && h0 + i < nh) {
      r[i][0].load(src + (h0 + i) * HD + d0);
      r[i][1].load(src + (h0 + i) * HD + d1);
    }
  // the angles of its 8 pairs (d0 + i, d1 + i), or of 4 neighbours' pairs in each chunk, and its 16 weights
  float4 cs[2], sn[2], w[4];
  if (live && turns) {
    const int i0 = INTER ? d0 / 2 : d0, i1 = INTER ? d1 / 2 : d0 + 4;
    const float *ct = a.cos_t + (int64_t)pos * half, *st = a.sin_t + (int64_t)pos * half;
    cs[0] = *reinterpret_cast<const float4*>(ct + i0); cs[1] = *reinterpret_cast<const float4*>(ct + i1);
    sn[0] = *reinterpret_cast<const float4*>(st + i0); sn[1] = *reinterpret_cast<const float4*>(st + i1);
  }
  const float* nw = is_q ? a.q_norm : a.k_norm;
  if (nw) {
    w[0] = reinterpret_cast<const float4*>(nw + d0)[0]; w[1] = reinterpret_cast<const float4*>(nw + d0)[1];
    w[2] = reinterpret_cast<const float4*>(nw + d1)[0]; w[3] = reinterpret_cast<const float4*>(nw + d1)[1];
  }
  const float *c = reinterpret_cast<const float*>(cs), *s = reinterpret_cast<const float*>(sn), *ww = reinterpret_cast<const float*>(w);
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    if (h0 + i >= nh) break;             // the same for the lanes of a head
    float x[2][8];
    r[i][0].get(x[0]);
    r[i][1].get(x[1]);
    if (nw) {
      float ss[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) { ss[0] = fmaf(x[0][j], x[0][j], ss[0]); ss[1] = fmaf(x[1][j], x[1][j], ss[1]); }
      float sum = ss[0] + ss[1];
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
      const float inv = rsqrtf(sum * (1.0f / HD) + a.eps);   // off by 2 units of 2^-24 or so
#pragma unroll
      for (int j = 0; j < 8; ++j) { x[0][j] = x[0][j] * inv * ww[j]; x[1][j] = x[1][j] * inv * ww[8 + j]; }
    }
    if (turns) {
      if (INTER) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float u = x[q][2 * j], v = x[q][2 * j + 1], co = c[4 * q + j], si = s[4 * q + j];
            x[q][2 * j] = u * co - v * si;
            x[q][2 * j + 1] = v * co + u * si;
          }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = x[0][j], v = x[1][j];
          x[0][j] = u * c[j] - v * s[j];
          x[1][j] = v * c[j] + u * s[j];
        }
      }
    }
    if (live) {
      store8(dst + (h0 + i) * HD + d0, x[0]);
      store8(dst + (h0 + i) * HD + d1, x[1]);
    }
  }
}

// Any even head_dim up to 512, any even rot_dim, any alignment: one warp per head, through shared memory.
template <class TI, class TO>
__global__ void __launch_bounds__(kThreads) qk_rope_any_kernel(const ms_qk_rope a, uint32_t* err) {
  __shared__ float sh[kThreads / 32][512];
  const int lane = threadIdx.x & 31, hd = a.head_dim, half = a.rot_dim / 2;
  float* x = sh[threadIdx.x >> 5];
  const uint32_t item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), nh = a.heads + a.kv_heads;
  const uint32_t t = item / nh;
  const int hh = item % nh;
  pdl_wait_prior();
  pdl_launch_dependents();
  if (t >= (uint32_t)a.n_tokens) return;
  const int pos = a.pos[t];
  if (pos < 0 || pos >= a.max_pos) {
    if (hh == 0 && lane == 0) atomicOr(err, EF_BAD_INDEX);
    return;
  }
  const bool is_q = hh < a.heads;
  const int h = is_q ? hh : hh - a.heads;
  const TI* src = (const TI*)(is_q ? a.q : a.k) + (int64_t)t * (is_q ? a.q_stride : a.k_stride) + h * hd;
  TO* dst = (TO*)(is_q ? a.q_out : a.k_out) + (int64_t)t * (is_q ? a.q_out_stride : a.k_out_stride) + h * hd;
  float ss = 0.f;
  for (int i = lane; i < hd; i += 32) {
    const float v = to_f32(src[i]);
    x[i] = v;
    ss = fmaf(v, v, ss);
  }
  const float* nw = is_q ? a.q_norm : a.k_norm;
  __syncwarp();
  if (nw) {
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)hd + a.eps);
    for (int i = lane; i < hd; i += 32) x[i] *= inv * nw[i];
    __syncwarp();
  }
  for (int i = lane; i < half; i += 32) {
    const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
    const float u = x[i0], v = x[i1], c = a.cos_t[(int64_t)pos * half + i], s = a.sin_t[(int64_t)pos * half + i];
    x[i0] = u * c - v * s;
    x[i1] = v * c + u * s;
  }
  __syncwarp();
  for (int i = lane; i < hd; i += 32) dst[i] = from_f32<TO>(x[i]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class TI, class TO, int LPR, int HPG>
void start_vec(const DevCtx& c, const ms_qk_rope& a, cudaStream_t s) {
  const uint32_t nb = (a.heads + HPG - 1) / HPG + (a.kv_heads + HPG - 1) / HPG;
  const uint32_t grid = ((uint64_t)a.n_tokens * nb + kThreads / LPR - 1) / (kThreads / LPR);
  if (a.interleaved) launch_early(qk_rope_kernel<TI, TO, LPR, HPG, true>, c.sm_count, grid, kThreads, s, a, c.err);
  else launch_early(qk_rope_kernel<TI, TO, LPR, HPG, false>, c.sm_count, grid, kThreads, s, a, c.err);
}

template <class TI, class TO>
void start(const DevCtx& c, const ms_qk_rope& a, cudaStream_t s) {
  const int hd = a.head_dim;
  const bool vec = (hd == 64 || hd == 128 || hd == 256) && a.rot_dim % 16 == 0 && a.q_stride % 8 == 0 &&
                   a.k_stride % 8 == 0 && a.q_out_stride % 8 == 0 && a.k_out_stride % 8 == 0 && aligned16(a.q) &&
                   aligned16(a.k) && aligned16(a.q_out) && aligned16(a.k_out) && aligned16(a.cos_t) && aligned16(a.sin_t) &&
                   aligned16(a.q_norm) && aligned16(a.k_norm);
  if (!vec) {
    const uint64_t items = (uint64_t)a.n_tokens * (a.heads + a.kv_heads);
    launch_early(qk_rope_any_kernel<TI, TO>, c.sm_count, (uint32_t)((items + kThreads / 32 - 1) / (kThreads / 32)), kThreads, s, a, c.err);
    return;
  }
  // Four heads per group share a look-up and the table's row; with few rows one, so that the loads spread over the
  // SMs.  32 + 4 heads of 128 dims, four against one: 2.3 / 1.6 us (1 token), 2.5 / 1.8 (32), 2.7 / 2.7 (256),
  // 4.6 / 6.1 (1,024), 12.6 / 17.6 (4,096).
  const bool wide = (int64_t)a.n_tokens * (a.heads + a.kv_heads) * hd / 16 >= (int64_t)c.sm_count * 512;
  if (hd == 64) wide ? start_vec<TI, TO, 4, 4>(c, a, s) : start_vec<TI, TO, 4, 1>(c, a, s);
  else if (hd == 128) wide ? start_vec<TI, TO, 8, 4>(c, a, s) : start_vec<TI, TO, 8, 1>(c, a, s);
  else wide ? start_vec<TI, TO, 16, 4>(c, a, s) : start_vec<TI, TO, 16, 1>(c, a, s);
}

template <class TI>
void start_out(const DevCtx& c, const ms_qk_rope& a, cudaStream_t s) {
  if (a.out_type == MS_Q_F32) start<TI, float>(c, a, s);
  else if (a.out_type == MS_Q_F16) start<TI, __half>(c, a, s);
  else start<TI, __nv_bfloat16>(c, a, s);
}

}  // namespace

cudaError_t launch_qk_rope(const DevCtx& c, const ms_qk_rope& a, cudaStream_t s) {
  if (a.n_tokens == 0) return cudaSuccess;
  if (a.in_type == MS_Q_F32) start_out<float>(c, a, s);
  else if (a.in_type == MS_Q_F16) start_out<__half>(c, a, s);
  else start_out<__nv_bfloat16>(c, a, s);
  return cudaGetLastError();
}

}  // namespace ms
