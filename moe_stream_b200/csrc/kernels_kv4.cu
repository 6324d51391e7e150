// kernels_kv4.cu — the paged 4-bit K/V cache: quantising rows into it and reading them back.
//
// A group of 32 dims keeps d = f16((max - min) / 15), o = f16(min - 16 d) and 4-bit codes c that stand for
// o + d (16 + c).  The hidden 16 makes a code the top mantissa bits of the f16 or bf16 number 16 + c, so the
// attention kernel builds tensor-core operands from it with one mask-and-or.  The layout of a block of 16 tokens
// is in include/moestream_cuda.h.  Both kernels are bound by memory: every row and every block byte moves once.
// Reading 57,200 tokens of 4 heads of 128 dims (154 MB) takes 29 us, 5.3 TB/s, writing them 46 us, 3.3 TB/s (instructions of
// the quantiser); writing 8,925 tokens of 8 heads of 64 dims (24 MB) takes 10.7 us, most of it latency, and reading them back 6.5.
#include <type_traits>

#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace ms {
namespace {

constexpr int kThreads = 128, kRows = 16;   // rows of a block at most

// ---- which rows of the block lead a token pair of the cache (an even token, or the first row of a sequence), and where
// their pair stands.  A pair's V codes share words, so the lanes that hold both tokens store whole words.  One
// thread looks up a row for all heads. ----
struct Leads {
  int64_t block[kRows];   // the 16-token block of head 0, counted in blocks from the start of the pages
  int row[kRows];
  int tok[kRows];         // token in the block; + 16: the next row is the pair's other token
  int n;
};
__device__ __forceinline__ void find_leads(const ms_kv4_cache& c, const ms_kv4_rows& r, int rows, Leads& ls, uint32_t* err) {
  pdl_wait_prior();
  pdl_launch_dependents();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, j = blockIdx.x * rows + lane;
    bool lead = false;
    int64_t block = 0;
    int tok = 0;
    // the row's sequence, the last one that begins at or before it: from 32 samples of the offsets, one load, and among
    // the sequences between two of them by bisection
    const int stride = (c.n_seqs - 1) / 32 + 1, mine = lane * stride;
    const bool have = mine < c.n_seqs;
    const int lo = have ? r.cu[mine] : 0x7fffffff, hi = have && stride == 1 ? r.cu[mine + 1] : 0, st = have && stride == 1 ? r.start[mine] : 0;
    int i = 0;
    if (c.n_seqs > 1)
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (__shfl_sync(0xffffffffu, lo, i + step) <= j) i += step;
    int begin = __shfl_sync(0xffffffffu, lo, i), end = __shfl_sync(0xffffffffu, hi, i), first = __shfl_sync(0xffffffffu, st, i);
    if (stride > 1 && lane < rows) {
      i *= stride;
      for (int last = min(i + stride, c.n_seqs) - 1; i < last;) {
        const int mid = (i + last + 1) >> 1;
        if (r.cu[mid] <= j) i = mid;
        else last = mid - 1;
      }
      begin = r.cu[i]; end = r.cu[i + 1]; first = r.start[i];
    }
    if (j < begin || j >= end) i = -1;     // behind the last sequence
    if (lane < rows && j < r.total) {
      if (i >= 0) {
        const int at = j - begin, pos = first + at;
        if (!(pos & 1) || at == 0) {
          block = kv4_block(c, i, pos, 0);
          lead = block >= 0;
          if (!lead) atomicOr(err, EF_BAD_INDEX);
          tok = (pos & 15) | (!(pos & 1) && j + 1 < end && j + 1 < r.total ? 16 : 0);
        }
      }
    }
    const unsigned mask = __ballot_sync(0xffffffffu, lead);
    if (lead) {
      const int k = __popc(mask & ((1u << lane) - 1));
      ls.block[k] = block;
      ls.row[k] = j;
      ls.tok[k] = tok;
    }
    if (lane == 0) ls.n = __popc(mask);
  } else if (threadIdx.x < 64) {           // the second warps of all blocks look the offsets over together
    if (!offsets_ok(r.cu, c.n_seqs, r.total, blockIdx.x * 32, gridDim.x * 32)) atomicOr(err, EF_BAD_INDEX);
  }
  __syncthreads();
}

// ---- quantising: 8 dims of a group of 32 held by 4 neighbouring lanes (all lanes of a warp take part) ----
// largest value and minus the smallest of two packed pairs' halves; NaN when there is one
template <class T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <class T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void range_of(const float (&x)[8], float& lo, float& hi) {
  lo = fminf(min3(x[0], x[1], x[2]), min3(min3(x[3], x[4], x[5]), x[6], x[7]));
  hi = fmaxf(max3(x[0], x[1], x[2]), max3(max3(x[3], x[4], x[5]), x[6], x[7]));
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
}
// smallest and largest value of the group.  False when one of its values is beyond +-16384, infinite or NaN
template <class T>
__device__ __forceinline__ bool range_of(const Raw8<T>& raw, const float (&)[8], float& lo, float& hi) {
  const uint32_t a = max2<T>(max2<T>(raw.u.x, raw.u.y), max2<T>(raw.u.z, raw.u.w));
  const uint32_t b = min2<T>(min2<T>(raw.u.x, raw.u.y), min2<T>(raw.u.z, raw.u.w)) ^ 0x80008000u;
  uint32_t m = max2<T>(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
  m = max2<T>(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max2<T>(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const float2 f = unpack2<T>(m);
  hi = f.x;
  lo = -f.y;
  return hi <= 16384.f && lo >= -16384.f;
}
__device__ __forceinline__ bool range_of(const Raw8<float>&, const float (&x)[8], float& lo, float& hi) {
  range_of(x, lo, hi);
  float sum = 0.f;                         // NaN when one is
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf(x[i], 0.f, sum);
  return hi <= 16384.f && lo >= -16384.f && sum == 0.f;
}
struct Group8 {
  uint32_t scale;   // f16 d, f16 o
  uint64_t t[4];    // the codes as pairs of f32
};
constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: adding it rounds to an integer in the low bits
// The kernel executes 142 warp instructions for 8 values of each lane; with the values one by one and __fdiv_rn it were 201,
// which bound it (write and read back 8,925 tokens of 8 heads of 64 dims: 19.0 us for 17.0).
template <class T>
__device__ __forceinline__ Group8 quantise8(const Raw8<T>& raw) {
  Group8 g;
  float x[8], lo, hi;
  raw.get(x);
  if (__any_sync(0xffffffffu, !range_of(raw, x, lo, hi))) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -16384.f), 16384.f);
    range_of(x, lo, hi);
  }
  // d and o are rounded to f16 first and the codes computed from the rounded values.  The division by 15 is the product
  // with its rounded reciprocal and Markstein's correction, which rounds it correctly (true for each of the 2^23 significands)
  constexpr float k15 = 1.f / 15.f;
  const float span = __fsub_rn(hi, lo), q = __fmul_rn(span, k15);
  const __half dh = __float2half_rn(fmaf(fmaf(-15.f, q, span), k15, q));
  const float d = __half2float(dh);
  const __half oh = __float2half_rn(fmaf(-16.f, d, lo));     // 16 d is exact
  const float o = __half2float(oh);
  g.scale = __half_as_ushort(dh) | (uint32_t)__half_as_ushort(oh) << 16;
  // rint((x - o) / d) - 16, clamped to 0 .. 15, as the fifteenfold of a value clamped to 0 .. 1, by an approximate
  // reciprocal: together off by less than 2^-16 here.  Within 2^-12 of a tie, by the division
  float rd;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rd) : "f"(d));
  rd = d > 0.f ? rd * k15 : 0.f;
  const uint64_t o2 = pair(-o, -o), up = pair(kMagic, kMagic), down = pair(-kMagic, -kMagic), p15 = pair(15.f, 15.f), n15 = pair(-15.f, -15.f);
  float near = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpair(add2(pair(x[2 * i], x[2 * i + 1]), o2));
    const uint64_t y = pair(__saturatef(fmaf(v.x, rd, -16.f * k15)), __saturatef(fmaf(v.y, rd, -16.f * k15)));
    g.t[i] = add2(fma2(y, p15, up), down);
    const float2 e = unpair(fma2(y, n15, g.t[i]));
    near = max3(near, fabsf(e.x), fabsf(e.y));
  }
  if (near > 0.5f - 0x1p-12f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) t[e] = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[2 * i + e], o), d)) - 16.0f, 0.f), 15.f);
      g.t[i] = pair(t[0], t[1]);
    }
  }
  return g;
}
// codes 2 n + h at bits 4 n + 16 h
__device__ __forceinline__ uint32_t k_word(const Group8& g) {
  const uint64_t k16 = pair(16.f, 16.f);
  const float2 w = unpair(add2(fma2(fma2(fma2(g.t[3], k16, g.t[2]), k16, g.t[1]), k16, g.t[0]), pair(kMagic, kMagic)));
  return __byte_perm(__float_as_uint(w.x), __float_as_uint(w.y), 0x5410);
}
// codes 4 q .. 4 q + 3 in the low 16 bits
template <int Q>
__device__ __forceinline__ uint32_t v_quad(const Group8& g) {
  const float2 w = unpair(fma2(g.t[2 * Q + 1], pair(256.f, 256.f), g.t[2 * Q]));
  return __float_as_uint(fmaf(w.y, 16.f, w.x) + kMagic);
}

// A row's heads are laid over the threads in order, 8 dims a thread, so a block's threads run through its rows.
template <class T, int HD>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const ms_kv4_cache c, const ms_kv4_rows r, int rows, uint32_t* err) {
  constexpr int LPR = HD / 8, G = HD / 32;
  __shared__ Leads ls;
  find_leads(c, r, rows, ls, err);
  const int width = c.kv_heads * LPR, n = ls.n, per_head = c.page_tokens / 16;
  int k = 0, at = threadIdx.x;
  while (at >= width) { at -= width; ++k; }
  for (int b = 0; b < n * width; b += kThreads) {          // the same count for all threads: the lanes exchange minima
    const bool live = k < n;
    const int tk = live ? ls.tok[k] : 0, row = live ? ls.row[k] : 0;
    const bool two = tk & 16;
    const int64_t at_k = (int64_t)row * r.k_stride + at * 8, at_v = (int64_t)row * r.v_stride + at * 8;
    Raw8<T> kr[2], vr[2];
    kr[0].zero(); kr[1].zero(); vr[0].zero(); vr[1].zero();
    if (live) {
      kr[0].load((const T*)r.k + at_k);
      vr[0].load((const T*)r.v + at_v);
      if (two) {
        kr[1].load((const T*)r.k + at_k + r.k_stride);
        vr[1].load((const T*)r.v + at_v + r.v_stride);
      }
    }
    const int head = at / LPR, part = at % LPR, w = part >> 2, t = part & 3, tok = tk & 15, pair = tok >> 1;
    uint8_t* blk = (uint8_t*)c.pages + ((live ? ls.block[k] : 0) + (int64_t)head * per_head) * kv4_block_bytes(HD);
    uint32_t* ks = reinterpret_cast<uint32_t*>(blk + kv4_k_scales(HD)) + tok * G + w;
    uint32_t* kc = reinterpret_cast<uint32_t*>(blk) + tok * 4 * G + t * G + w;
    {
      const Group8 g = quantise8(kr[0]);
      if (live) {
        *kc = k_word(g);
        if (t == 0) *ks = g.scale;
      }
    }
    const bool any_two = __any_sync(0xffffffffu, two);
    if (any_two) {
      const Group8 g = quantise8(kr[1]);
      if (live && two) {
        kc[4 * G] = k_word(g);
        if (t == 0) ks[G] = g.scale;
      }
    }
    const Group8 g0 = quantise8(vr[0]);
    // lanes 2 C and 2 C + 1 hold the quads 0, 1 and 2, 3 of chunk C
    uint16_t* vc = reinterpret_cast<uint16_t*>(blk + kv4_v_codes(HD)) + (pair * (HD / 16) + kv4_v_chunk<HD>(part >> 1, pair)) * 8 + (part & 1) * 4;
    uint16_t* vs = reinterpret_cast<uint16_t*>(blk + kv4_v_scales(HD)) + (pair * G + w) * 4;
    if (any_two) {
      const Group8 g1 = quantise8(vr[1]);
      if (live && two) {
        *reinterpret_cast<uint2*>(vc) = make_uint2(__byte_perm(v_quad<0>(g0), v_quad<0>(g1), 0x5410), __byte_perm(v_quad<1>(g0), v_quad<1>(g1), 0x5410));
        if (t == 0)
          *reinterpret_cast<uint2*>(vs) = make_uint2(__byte_perm(g0.scale, g1.scale, 0x5410), __byte_perm(g0.scale, g1.scale, 0x7632));
      }
    }
    if (live && !two) {
      const int par = tok & 1;
      vc[par] = (uint16_t)v_quad<0>(g0);
      vc[2 + par] = (uint16_t)v_quad<1>(g0);
      if (t == 0) {
        vs[par] = (uint16_t)g0.scale;
        vs[2 + par] = (uint16_t)(g0.scale >> 16);
      }
    }
    at += kThreads;
    while (at >= width) { at -= width; ++k; }
  }
}

// nibble N of a word as the f32 number 16 + c: the code in the mantissa bits of 16 that weigh 1 to 8
template <int N>
__device__ __forceinline__ float code_f32(uint32_t w) {
  constexpr int UP = 19 - 4 * N;
  return __uint_as_float(((UP >= 0 ? w << (UP >= 0 ? UP : 0) : w >> (UP < 0 ? -UP : 0)) & 0x00780000u) | 0x41800000u);
}
// values o + d (16 + c) of 8 codes; d (16 + c) is exact
__device__ __forceinline__ void k_values(uint32_t w, float d, float o, float (&x)[8]) {
  x[0] = fmaf(d, code_f32<0>(w), o); x[1] = fmaf(d, code_f32<4>(w), o);
  x[2] = fmaf(d, code_f32<1>(w), o); x[3] = fmaf(d, code_f32<5>(w), o);
  x[4] = fmaf(d, code_f32<2>(w), o); x[5] = fmaf(d, code_f32<6>(w), o);
  x[6] = fmaf(d, code_f32<3>(w), o); x[7] = fmaf(d, code_f32<7>(w), o);
}
template <int HALF>
__device__ __forceinline__ void v_values(uint2 w, float d, float o, float (&x)[8]) {
  constexpr int H = 4 * HALF;
  x[0] = fmaf(d, code_f32<H>(w.x), o); x[1] = fmaf(d, code_f32<H + 1>(w.x), o);
  x[2] = fmaf(d, code_f32<H + 2>(w.x), o); x[3] = fmaf(d, code_f32<H + 3>(w.x), o);
  x[4] = fmaf(d, code_f32<H>(w.y), o); x[5] = fmaf(d, code_f32<H + 1>(w.y), o);
  x[6] = fmaf(d, code_f32<H + 2>(w.y), o); x[7] = fmaf(d, code_f32<H + 3>(w.y), o);
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const ms_kv4_cache c, const ms_kv4_rows r, int rows, uint32_t* err) {
  constexpr int LPR = HD / 8, G = HD / 32;
  __shared__ Leads ls;
  find_leads(c, r, rows, ls, err);
  const int width = c.kv_heads * LPR, n = ls.n, per_head = c.page_tokens / 16;
  int k = 0, at = threadIdx.x;
  while (at >= width) { at -= width; ++k; }
#pragma unroll 2
  for (; k < n;) {
    const int tk = ls.tok[k], row = ls.row[k], head = at / LPR, part = at % LPR, w = part >> 2, t = part & 3, tok = tk & 15, pair = tok >> 1;
    const uint8_t* blk = (const uint8_t*)c.pages + (ls.block[k] + (int64_t)head * per_head) * kv4_block_bytes(HD);
    const uint32_t* kc = reinterpret_cast<const uint32_t*>(blk) + tok * 4 * G + t * G + w;
    const uint32_t* ks = reinterpret_cast<const uint32_t*>(blk + kv4_k_scales(HD)) + tok * G + w;
    const bool two = tk & 16;
    const uint32_t k0 = kc[0], s0 = ks[0], k1 = two ? kc[4 * G] : 0u, s1 = two ? ks[G] : 0u;
    const uint2 vw = *reinterpret_cast<const uint2*>(blk + kv4_v_codes(HD) + (pair * (HD / 16) + kv4_v_chunk<HD>(part >> 1, pair)) * 16 + (part & 1) * 8);
    const uint2 vs = *reinterpret_cast<const uint2*>(blk + kv4_v_scales(HD) + (pair * G + w) * 8);
    T* kd = (T*)r.k + (int64_t)row * r.k_stride + at * 8;
    T* vd = (T*)r.v + (int64_t)row * r.v_stride + at * 8;
    const float2 vds = unpack2<__half>(vs.x), vos = unpack2<__half>(vs.y);
    float x[8];
    float2 s = unpack2<__half>(s0);
    k_values(k0, s.x, s.y, x);
    store8(kd, x);
    if (tok & 1) v_values<1>(vw, vds.y, vos.y, x);
    else v_values<0>(vw, vds.x, vos.x, x);
    store8(vd, x);
    if (two) {
      s = unpack2<__half>(s1);
      k_values(k1, s.x, s.y, x);
      store8(kd + r.k_stride, x);
      v_values<1>(vw, vds.y, vos.y, x);
      store8(vd + r.v_stride, x);
    }
    at += kThreads;
    while (at >= width) { at -= width; ++k; }
  }
}

template <class T, int HD>
cudaError_t start(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_rows& r, bool write, cudaStream_t s) {
  // 16 rows share a look-up, with few rows down to 2, so that a decode step spreads over the SMs (write and read back,
  // 16 rows against 2: 15.0 / 5.1 us for 32 tokens, 19.5 / 22.3 for 8,925, where the rule takes 8: 17.0)
  int rows = kRows;
  while (rows > 2 && (int64_t)r.total < (int64_t)rows * 4 * d.sm_count) rows /= 2;
  const uint32_t grid = (uint32_t)(((int64_t)r.total + rows - 1) / rows);
  if (write) launch_early(kv4_write_kernel<T, HD>, d.sm_count, grid, kThreads, s, c, r, rows, d.err);
  else launch_early(kv4_read_kernel<T, HD>, d.sm_count, grid, kThreads, s, c, r, rows, d.err);
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
