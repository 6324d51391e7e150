// kernels_kv4.cu — the paged 4-bit K/V cache: quantising rows into it and reading them back.
//
// A group of 32 dims keeps d = f16((max - min) / 15), o = f16(min - 16 d) and 4-bit codes c that stand for
// o + d (16 + c).  The hidden 16 makes a code the top mantissa bits of the f16 or bf16 number 16 + c, so the
// attention kernel builds tensor-core operands from it with one mask-and-or.  The layout of a block of 16 tokens
// is in include/moestream_cuda.h.  Both kernels are bound by memory: every row and every block byte moves once.
#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace ms {
namespace {

constexpr int kThreads = 128;

// 8 dims of a group of 32 held by 4 neighbouring lanes -> codes and the group's scales
struct Group8 {
  float d, o;
  uint32_t c[8];
};
__device__ __forceinline__ Group8 quantise8(float (&x)[8]) {
  Group8 g;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -16384.f), 16384.f);
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
  // d and o are rounded to f16 first and the codes computed from the rounded values
  g.d = __half2float(__float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f)));
  g.o = __half2float(__float2half_rn(__fsub_rn(lo, 16.0f * g.d)));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = g.d > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[i], g.o), g.d)) - 16.0f : 0.f;
    g.c[i] = (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
  }
  return g;
}
__device__ __forceinline__ uint16_t half_bits(float x) { return __half_as_ushort(__float2half_rn(x)); }

// Which rows a group of hd / 8 lanes takes: of the packed rows 2 m and 2 m + 1 those that lead a token pair of
// the cache (an even token, or the first row of a sequence), each with its partner when that is a row too.  A
// pair's V codes share words, so a group that holds both tokens stores whole words.
struct Lead {
  int seq = -1, row, pos;
  bool two;   // the partner pos + 1 is row + 1
};
__device__ __forceinline__ Lead lead_of(const ms_kv4_rows& r, int n_seqs, int j) {
  Lead l;
  if (j >= r.total) return l;
  const int i = seq_of_row(r.cu, n_seqs, j);
  if (i < 0) return l;
  const int at = j - r.cu[i], pos = r.start[i] + at;
  if ((pos & 1) && at > 0) return l;
  l.seq = i;
  l.row = j;
  l.pos = pos;
  l.two = !(pos & 1) && j + 1 < r.cu[i + 1] && j + 1 < r.total;
  return l;
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const ms_kv4_cache c, const ms_kv4_rows r, uint32_t* err) {
  constexpr int LPR = HD / 8, G = HD / 32;
  const int part = threadIdx.x % LPR, w = part >> 2, t = part & 3;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int head = item % c.kv_heads;
  const int64_t m = item / c.kv_heads;
  for (int e = 0; e < 2; ++e) {
    Lead l;
    if (2 * m + e < r.total) l = lead_of(r, c.n_seqs, (int)(2 * m + e));
    uint8_t* blk = l.seq >= 0 ? kv4_block(c, l.seq, l.pos, head) : nullptr;
    if (l.seq >= 0 && !blk && part == 0) atomicOr(err, EF_BAD_INDEX);
    Group8 k[2], v[2];
    // every lane quantises (the shuffles need whole warps); lanes without a row work on zeros
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (blk && (p == 0 || l.two)) {
        Raw8<T> a, b;
        a.load((const T*)r.k + (int64_t)(l.row + p) * r.k_stride + head * HD + part * 8);
        b.load((const T*)r.v + (int64_t)(l.row + p) * r.v_stride + head * HD + part * 8);
        a.get(x);
        b.get(y);
      }
      k[p] = quantise8(x);
      v[p] = quantise8(y);
    }
    if (!blk) continue;
    const int tok = l.pos & 15, pair = tok >> 1;
    uint16_t vq[2][2];   // [token of the pair][quad]
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (p == 1 && !l.two) break;
      uint32_t word = 0;
#pragma unroll
      for (int n = 0; n < 4; ++n) word |= k[p].c[2 * n] << (4 * n) | k[p].c[2 * n + 1] << (4 * n + 16);
      reinterpret_cast<uint32_t*>(blk)[(tok + p) * 4 * G + t * G + w] = word;
      if (t == 0)
        reinterpret_cast<uint32_t*>(blk + kv4_k_scales(HD))[(tok + p) * G + w] =
            half_bits(k[p].d) | (uint32_t)half_bits(k[p].o) << 16;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        vq[p][q] = (uint16_t)(v[p].c[4 * q] | v[p].c[4 * q + 1] << 4 | v[p].c[4 * q + 2] << 8 | v[p].c[4 * q + 3] << 12);
    }
    // lanes 2 C and 2 C + 1 hold the quads 0, 1 and 2, 3 of chunk C
    uint16_t* vc = reinterpret_cast<uint16_t*>(blk + kv4_v_codes(HD)) + (pair * (HD / 16) + kv4_v_chunk<HD>(part >> 1, pair)) * 8 + (part & 1) * 4;
    uint16_t* vs = reinterpret_cast<uint16_t*>(blk + kv4_v_scales(HD)) + (pair * G + w) * 4;
    if (l.two) {
      *reinterpret_cast<uint2*>(vc) = make_uint2(vq[0][0] | (uint32_t)vq[1][0] << 16, vq[0][1] | (uint32_t)vq[1][1] << 16);
      if (t == 0)
        *reinterpret_cast<uint2*>(vs) = make_uint2(half_bits(v[0].d) | (uint32_t)half_bits(v[1].d) << 16,
                                                   half_bits(v[0].o) | (uint32_t)half_bits(v[1].o) << 16);
    } else {
      const int par = tok & 1;
      vc[par] = vq[0][0];
      vc[2 + par] = vq[0][1];
      if (t == 0) {
        vs[par] = half_bits(v[0].d);
        vs[2 + par] = half_bits(v[0].o);
      }
    }
  }
}

// the 4 codes of a 16-bit quad -> values
__device__ __forceinline__ void quad_values(uint32_t u, float d, float o, float* x) {
#pragma unroll
  for (int n = 0; n < 4; ++n) x[n] = fmaf(d, (float)(16 + ((u >> (4 * n)) & 15u)), o);   // d * (16 + c) is exact
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const ms_kv4_cache c, const ms_kv4_rows r, uint32_t* err) {
  constexpr int LPR = HD / 8, G = HD / 32;
  const int part = threadIdx.x % LPR, w = part >> 2, t = part & 3;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int head = item % c.kv_heads;
  const int64_t m = item / c.kv_heads;
  for (int e = 0; e < 2; ++e) {
    if (2 * m + e >= r.total) return;
    const Lead l = lead_of(r, c.n_seqs, (int)(2 * m + e));
    if (l.seq < 0) continue;
    const uint8_t* blk = kv4_block(c, l.seq, l.pos, head);
    if (!blk) {
      if (part == 0) atomicOr(err, EF_BAD_INDEX);
      continue;
    }
    const int tok = l.pos & 15, pair = tok >> 1;
    const uint2 vw = *reinterpret_cast<const uint2*>(blk + kv4_v_codes(HD) + (pair * (HD / 16) + kv4_v_chunk<HD>(part >> 1, pair)) * 16 + (part & 1) * 8);
    const uint2 vs = *reinterpret_cast<const uint2*>(blk + kv4_v_scales(HD) + (pair * G + w) * 8);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (p == 1 && !l.two) break;
      const uint32_t kw = reinterpret_cast<const uint32_t*>(blk)[(tok + p) * 4 * G + t * G + w];
      const float2 ks = unpack2<__half>(reinterpret_cast<const uint32_t*>(blk + kv4_k_scales(HD))[(tok + p) * G + w]);
      float x[8], y[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        x[2 * n] = fmaf(ks.x, (float)(16 + ((kw >> (4 * n)) & 15u)), ks.y);
        x[2 * n + 1] = fmaf(ks.x, (float)(16 + ((kw >> (4 * n + 16)) & 15u)), ks.y);
      }
      const int sh = ((tok + p) & 1) * 16;
      const float vd = h2f_bits((uint16_t)(vs.x >> sh)), vo = h2f_bits((uint16_t)(vs.y >> sh));
      quad_values((vw.x >> sh) & 0xFFFFu, vd, vo, y);
      quad_values((vw.y >> sh) & 0xFFFFu, vd, vo, y + 4);
      store8((T*)r.k + (int64_t)(l.row + p) * r.k_stride + head * HD + part * 8, x);
      store8((T*)r.v + (int64_t)(l.row + p) * r.v_stride + head * HD + part * 8, y);
    }
  }
}

template <class T, int HD>
cudaError_t start(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_rows& r, bool write, cudaStream_t s) {
  const int64_t items = ((int64_t)r.total + 1) / 2 * c.kv_heads, per = kThreads / (HD / 8);
  const uint32_t grid = (uint32_t)((items + per - 1) / per);
  if (write) kv4_write_kernel<T, HD><<<grid, kThreads, 0, s>>>(c, r, d.err);
  else kv4_read_kernel<T, HD><<<grid, kThreads, 0, s>>>(c, r, d.err);
  return cudaGetLastError();
}

template <class T>
cudaError_t start_hd(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_rows& r, bool write, cudaStream_t s) {
  if (c.head_dim == 64) return start<T, 64>(d, c, r, write, s);
  if (c.head_dim == 128) return start<T, 128>(d, c, r, write, s);
  return start<T, 256>(d, c, r, write, s);
}

}  // namespace

cudaError_t launch_kv4_rows(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_rows& r, bool write, cudaStream_t s) {
  if (r.total == 0) return cudaSuccess;
  if (r.type == MS_Q_F32) return start_hd<float>(d, c, r, write, s);
  if (r.type == MS_Q_F16) return start_hd<__half>(d, c, r, write, s);
  return start_hd<__nv_bfloat16>(d, c, r, write, s);
}

}  // namespace ms
