// w4_linear.cuh -- a few rows of activations times INT4 weights with group-128
// scales:
//
//   y[r, n] = act( sum_g s[n, g] * sum_{i in g} c[n, i] x'[r, i]  +  b[n] )
//
// with c the codes -8..7 of a packed weight (uint8 [N, K/2], low nibble = even
// column), s its fp16 scales [N, K/128], and x' = x, or x rotated by
// H128 / sqrt(128) in each group when the weight was (a ConvRot weight).  The
// activations are not quantised.
//
// Bound by the weight bytes, N K / 2: each is used by one row (or a few), and
// the kernel's whole work is to keep enough of them in flight.
//
// w4_prepare_kernel turns the rows into the matrix product's operand:
// rotated in fp32, scaled by a power of two per (row, group) that brings the
// group's largest value into [2^14, 2^15), and rounded to fp16.  The rounding
// is relative to the value for everything within 2^28 of the group's maximum,
// so it costs a rotated row up to 2^-11 (a bf16 rounding would cost 2^-8, as much
// as the output's), and an unrotated bf16 or fp16 row nothing.
//
// w4_linear_kernel: a warp takes 16 weight rows (the product's M) and a
// contiguous range of groups, straight from the checkpoint's layout: lane
// (r, t) loads the 32 codes 32 t.. of rows r and r + 8 with one 16-byte load
// each.  The k order inside a matrix product is free, so its 8 codes per
// 32-bit word become two k16 steps without any exchange; x' is laid out for
// that order by the prepare kernel, one 16-byte load per word, which L1 serves
// to the CTA's other warps.  Codes become fp16 exactly by setting the exponent
// of 1024 around a nibble.  Each group's sum is scaled by s and the row's
// power of two in fp32 and added up in fp32.  Two bursts of neighbouring groups
// are in flight per warp.  Where there are too few row tiles to fill the GPU, up
// to eight warps share a tile along k and add up in a fixed order.
//
// Measured: 36864 x 6144 (117 MB) by 1 row 31.5 us, 3.7 TB/s; by 8 rows 33.1;
// by 16 rows 43; 1536 x 2560 by 77 rows 8.1.  What is left over the loads' own
// 23 us are dequantisation and products that 16 warps do not hide entirely.
#pragma once
#include "elem16.cuh"

namespace k2b {

constexpr int W4_THREADS = 256;
constexpr int W4_WARPS = W4_THREADS / 32;
enum W4Act : int { W4_NONE = 0, W4_GELU = 1, W4_SILU = 2 };

// x' of 8 rows and one group: 4 words of 8 columns x 8 rows x 4 column quarters
constexpr int W4_FRAG_BYTES = 8 * 128 * 2;
inline long long w4_row_blocks(int m) { return (m + 7) / 8; }
inline long long w4_workspace_bytes(int m, int k) {
  return w4_row_blocks(m) * (k / 128) * (W4_FRAG_BYTES + 8 * (long long)sizeof(float));
}

// Whether the product kernel prepares its rows itself, in shared memory: a few
// rows of few groups, which a CTA does in less time than a second launch takes
// (one row by 6144 x 256: 3.1 against 4.0 us, with the host side of the call 5.8
// against 9.4).
constexpr int W4_FUSED_GROUPS = 16, W4_FUSED_ITEMS = 64;
inline bool w4_fused(int m, int k) {
  return m <= 8 && k <= 128 * W4_FUSED_GROUPS && (long long)m * (k / 128) <= W4_FUSED_ITEMS;
}

// x' of one (row, group) by a warp, to place `at` (the group's of the row's
// block of 8) of frag and factor; a row at or past m is zero.
template <typename T, bool ROTATE>
__device__ __forceinline__ void w4_prepare(const T* x, long long x_stride, uint8_t* frag, float* factor, int m, int row,
                                           int g, long long at) {
  const int lane = threadIdx.x & 31;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < m) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(x + row * x_stride + g * 128 + lane * 4));
    const float2 a = Elem16<T>::unpack(u.x), b = Elem16<T>::unpack(u.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  float scale = ROTATE ? kHadamardScale : 1.0f;  // what v still has to be multiplied by
  if (ROTATE) {
    // 128 terms of more than 2^120 could leave fp32 before they are scaled
    const float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    if (__any_sync(0xffffffffu, most > 1.329227995784916e36f)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= 0.00390625f;
      scale *= 256.0f;
    }
    const float a = v[0] + v[1], b = v[0] - v[1], c = v[2] + v[3], d = v[2] - v[3];
    v[0] = a + c, v[1] = b + d, v[2] = a - c, v[3] = b - d;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, v[i], o);
        v[i] = (lane & o) ? other - v[i] : v[i] + other;
      }
    }
  }
  // the largest finite magnitude sets the power of two
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = fabsf(v[i]);
    if (a <= 3.4028234663852886e38f) top = fmaxf(top, a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // exponent of 2^(14 - floor(log2 top)), kept inside the normal range
  int e = 127 + 14 - ((int)(__float_as_uint(top) >> 23) - 127);
  e = top > 0.0f ? min(max(e, 1), 253) : 127;
  const float up = __uint_as_float((uint32_t)e << 23), down = __uint_as_float((uint32_t)(254 - e) << 23);
  uint32_t lo = Elem16<__half>::pack(v[0] * up, v[1] * up), hi = Elem16<__half>::pack(v[2] * up, v[3] * up);
  // word order (0,4)(1,5)(2,6)(3,7): even lanes hold columns 0..3 of a word, odd lanes 4..7
  const uint32_t olo = __shfl_xor_sync(0xffffffffu, lo, 1), ohi = __shfl_xor_sync(0xffffffffu, hi, 1);
  uint2 out;
  if (lane & 1) {
    out = make_uint2(__byte_perm(ohi, hi, 0x5410), __byte_perm(ohi, hi, 0x7632));
  } else {
    out = make_uint2(__byte_perm(lo, olo, 0x5410), __byte_perm(lo, olo, 0x7632));
  }
  const int t = lane >> 3, word = (lane >> 1) & 3;
  *reinterpret_cast<uint2*>(frag + at * W4_FRAG_BYTES + ((word * 8 + (row & 7)) * 4 + t) * 16 + (lane & 1) * 8) = out;
  // 1/sqrt(128) of the rotation joins the factor
  if (lane == 0) factor[at * 8 + (row & 7)] = down * scale;
}

// One warp per (row, group); rows past m up to a whole block of 8 are zero.
template <typename T, bool ROTATE>
__global__ void __launch_bounds__(W4_THREADS)
    w4_prepare_kernel(const T* x, long long x_stride, uint8_t* frag, float* factor, int m, int groups, int total) {
  pdl_launch_dependents();
  const int item = blockIdx.x * W4_WARPS + (threadIdx.x >> 5);
  if (item >= total) return;
  const int row = item / groups, g = item % groups;
  w4_prepare<T, ROTATE>(x, x_stride, frag, factor, m, row, g, (long long)(row >> 3) * groups + g);
}

// Eight INT4 codes (two's complement nibbles, code i in bits 4i..) -> fp16
// pairs (0,4) (1,5) (2,6) (3,7).  Nibble ^ 8 is code + 8; under the exponent
// of 1024 it reads 1024 + (code + 8), and 16 times that for the odd nibbles.
__device__ __forceinline__ void w4_codes(uint32_t w, uint32_t (&h)[4]) {
  const __half2 one = __floats2half2_rn(1032.0f, 1032.0f);
  const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f), off = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = i ? w >> 8 : w;
    const uint32_t a = (u & 0x000F000Fu) ^ 0x64086408u, b = (u & 0x00F000F0u) ^ 0x64806480u;
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), one);
    const __half2 hb = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, off);
    h[2 * i] = *reinterpret_cast<const uint32_t*>(&ha);
    h[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hb);
  }
}

__device__ __forceinline__ float w4_act(float y, int act) {
  if (act == W4_GELU) return 0.5f * y * (1.0f + tanhf(0.7978845608028654f * (y + 0.044715f * y * y * y)));
  if (act == W4_SILU) return y / (1.0f + expf(-y));
  return y;
}

struct W4Params {
  const void* x;         // the rows themselves (a fused launch)
  long long x_stride;
  const uint8_t* w;      // [n, k/2]
  const unsigned short* scales;  // fp16 [n, groups]
  const uint8_t* frag;   // prepared rows (not a fused launch)
  const float* factor;
  const void* bias;      // [n] or null
  void* out;             // [m, n]
  int m, n, groups, act;
  int kw;                // warps of a CTA along k (1, 2, 4, 8); the others take further rows
};

// NT: blocks of 8 activation rows of this CTA (blockIdx.y * NT first), 1 or 2.
// FUSED: the CTA prepares the rows itself, with ROTATE or without.
template <typename T, int NT, bool FUSED = false, bool ROTATE = false>
__global__ void __launch_bounds__(W4_THREADS, 2) w4_linear_kernel(const __grid_constant__ W4Params p) {
  // Two bursts of BURST groups per warp: a burst asks for BURST x 64
  // neighbouring bytes of each row at once.  (Asked for group by group, five in
  // flight, the loads alone took 27 us of 36864 x 6144 instead of 23.  Bursts
  // of 3 and 4 cost more in registers than they give: 33 and 41 against 31 us
  // for the whole product.)
  constexpr int BURST = 2;
  __shared__ float red[W4_WARPS][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int kw = p.kw, rw = W4_WARPS / kw;
  const int wk = warp % kw, wr = warp / kw;
  const int per = (p.groups + kw - 1) / kw;
  const int g0 = wk * per, count = min(per, p.groups - g0);  // (may be none)
  const long long row_bytes = (long long)p.groups * 64;
  const int block0 = blockIdx.y * NT, mblocks = (p.m + 7) / 8;
  const int n0 = blockIdx.x * 16 * rw;  // the CTA's first weight row
  const int ra = min(n0 + wr * 16 + r, p.n - 1), rb = min(n0 + wr * 16 + r + 8, p.n - 1);

  uint4 wa[2][BURST], wb[2][BURST];
  uint32_t sa[2][BURST], sb[2][BURST];  // fp16 scales, a register each
  const uint8_t* pa = p.w + ra * row_bytes + g0 * 64 + t * 16;
  const uint8_t* pb = p.w + rb * row_bytes + g0 * 64 + t * 16;
  const unsigned short* qa = p.scales + (long long)ra * p.groups + g0;
  const unsigned short* qb = p.scales + (long long)rb * p.groups + g0;
  // burst u of the pair that starts at the pointers, `left` groups remaining there
  auto load = [&](int u, int left) {
#pragma unroll
    for (int s = 0; s < BURST; ++s)
      if (u * BURST + s < left) {
        wa[u][s] = ldg_stream(pa + (u * BURST + s) * 64);
        wb[u][s] = ldg_stream(pb + (u * BURST + s) * 64);
      }
#pragma unroll
    for (int s = 0; s < BURST; ++s)
      if (u * BURST + s < left) {
        sa[u][s] = ldg_ahead_u16(qa + u * BURST + s);
        sb[u][s] = ldg_ahead_u16(qb + u * BURST + s);
      }
  };
  load(0, count);
  load(1, count);
  const uint8_t* frag = p.frag;
  const float* factor = p.factor;
  if constexpr (FUSED) {
    __shared__ __align__(16) uint8_t own_frag[W4_FUSED_GROUPS * W4_FRAG_BYTES];
    __shared__ float own_factor[W4_FUSED_GROUPS * 8];
    for (int i = warp; i < p.m * p.groups; i += W4_WARPS) {
      const int row = i / p.groups, g = i - row * p.groups;
      w4_prepare<T, ROTATE>(static_cast<const T*>(p.x), p.x_stride, own_frag, own_factor, p.m, row, g, g);
    }
    __syncthreads();
    frag = own_frag;
    factor = own_factor;
  } else {
    pdl_wait();
  }

  // x' of row r of each block; rows past m are zero and are not read
  const uint8_t* px[NT];
  const float* pf[NT];
  bool live[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const long long at = (long long)min(block0 + i, mblocks - 1) * p.groups + g0;
    px[i] = frag + at * W4_FRAG_BYTES + lane * 16;
    pf[i] = factor + at * 8 + 2 * t;
    live[i] = (block0 + i) * 8 + r < p.m;
  }
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  for (int i0 = 0; i0 < count; i0 += 2 * BURST) {
    pa += 2 * BURST * 64;
    pb += 2 * BURST * 64;
    qa += 2 * BURST;
    qb += 2 * BURST;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int v = 0; v < BURST; ++v) {
        const int s = u * BURST + v;
        if (i0 + s >= count) break;
        const uint32_t ua[4] = {wa[u][v].x, wa[u][v].y, wa[u][v].z, wa[u][v].w};
        const uint32_t ub[4] = {wb[u][v].x, wb[u][v].y, wb[u][v].z, wb[u][v].w};
        float c[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t ha[4], hb[4];
          w4_codes(ua[w], ha);
          w4_codes(ub[w], hb);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (live[i]) x = *reinterpret_cast<const uint4*>(px[i] + s * W4_FRAG_BYTES + w * 512);
            mma16816<__half>(c[i], ha[0], hb[0], ha[1], hb[1], x.x, x.y);
            mma16816<__half>(c[i], ha[2], hb[2], ha[3], hb[3], x.z, x.w);
          }
        }
        const float fa = __half2float(__ushort_as_half((unsigned short)sa[u][v]));
        const float fb = __half2float(__ushort_as_half((unsigned short)sb[u][v]));
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float2 f = *reinterpret_cast<const float2*>(pf[i] + s * 8);
          // (the weight's scale first: the row's alone can take a sum out of fp32)
          acc[i][0] = fmaf(c[i][0] * fa, f.x, acc[i][0]);
          acc[i][1] = fmaf(c[i][1] * fa, f.y, acc[i][1]);
          acc[i][2] = fmaf(c[i][2] * fb, f.x, acc[i][2]);
          acc[i][3] = fmaf(c[i][3] * fb, f.y, acc[i][3]);
        }
      }
      load(u, count - i0 - 2 * BURST);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      px[i] += 2 * BURST * W4_FRAG_BYTES;
      pf[i] += 2 * BURST * 8;
    }
  }
  // the tile's sums over its kw warps, in warp order
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    red[warp][r][8 * i + 2 * t] = acc[i][0];
    red[warp][r][8 * i + 2 * t + 1] = acc[i][1];
    red[warp][r + 8][8 * i + 2 * t] = acc[i][2];
    red[warp][r + 8][8 * i + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  const int shift = kw == 8 ? 4 : kw == 4 ? 5 : kw == 2 ? 6 : 7;  // log2 of the CTA's weight rows
  const int rows = min(8 * NT, p.m - block0 * 8);
  for (int o = threadIdx.x; o < rows << shift; o += W4_THREADS) {
    const int nn = o & ((1 << shift) - 1), xr = o >> shift;
    if (n0 + nn < p.n) {
      float y = 0.0f;
      for (int q = 0; q < kw; ++q) y += red[(nn >> 4) * kw + q][nn & 15][xr];
      if (p.bias) y += Elem16<T>::to_float(static_cast<const T*>(p.bias)[n0 + nn]);
      static_cast<T*>(p.out)[(long long)(block0 * 8 + xr) * p.n + n0 + nn] = Elem16<T>::from_float(w4_act(y, p.act));
    }
  }
}

}  // namespace k2b
