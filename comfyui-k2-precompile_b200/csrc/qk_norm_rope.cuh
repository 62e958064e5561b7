// qk_norm_rope.cuh -- RMSNorm of every query and key head with the position
// rotation, one pass over q and one over k in the same launch.
//
//   y = R_pos (x * rsqrt(mean(x^2) + eps) * (w + 1)),   x one head of D values,
//
// R_pos the token's 2 x 2 matrices over the pairs (2i, 2i + 1) (freqs
// [.., L, D/2, 2, 2], or none).  All of it in fp32, rounded once when stored;
// the W4A4 projection's epilogue of the same operation rounds between its
// steps because the reference does.
//
// Bound by memory: 2 bytes read and 2 written per value, plus 8 D bytes of
// table per token.  D/8 lanes own a head (16 bytes each), so a warp takes
// 256 values at once; a warp's item is one token and QKN_HEADS heads, whose
// loads are all in flight before the first is used, and which share the
// token's table entries in registers.  The items of a token are neighbours,
// so the table comes from L1 after the first.
#pragma once
#include "elem16.cuh"

namespace k2b {

constexpr int QKN_HEADS = 8;     // heads per warp item
constexpr int QKN_THREADS = 256;

struct QkNormSide {
  const void* x;
  void* y;            // [B, L, heads, D] contiguous
  const float* w;     // [D], "w+1" form
  const float* freqs; // [fb, L, D/2, 2, 2] or null
  long long sb, sh, st;
  int length, heads, fb;
  float eps;
  long long items;    // batch * length * ceil(heads / QKN_HEADS)
};
struct QkNormParams {
  QkNormSide side[2];
};

template <typename T, int D>
__global__ void __launch_bounds__(QKN_THREADS) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int LPH = D / 8;               // lanes per head
  constexpr int HPS = 32 / LPH;            // heads per step
  constexpr int STEPS = QKN_HEADS / HPS;
  const int lane = threadIdx.x & 31;
  long long item = (long long)blockIdx.x * (QKN_THREADS / 32) + (threadIdx.x >> 5);
  const bool second = item >= p.side[0].items;
  if (second) item -= p.side[0].items;
  const QkNormSide& s = p.side[second ? 1 : 0];
  if (item >= s.items) return;
  const int chunks = (s.heads + QKN_HEADS - 1) / QKN_HEADS;
  const long long row = item / chunks;     // batch * length + token
  const int h0 = (int)(item % chunks) * QKN_HEADS + lane / LPH;
  const long long b = row / s.length, tok = row % s.length;
  const int c = (lane % LPH) * 8;          // this lane's first column

  const T* x = static_cast<const T*>(s.x) + b * s.sb + tok * s.st + c;
  uint4 v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    if (h0 + i * HPS < s.heads) v[i] = ldg_stream(x + (long long)(h0 + i * HPS) * s.sh);
  float w[8], f[16];
#pragma unroll
  for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(w + i) = __ldg(reinterpret_cast<const float4*>(s.w + c + i));
  if (s.freqs) {
    const float* fr = s.freqs + ((s.fb == 1 ? 0 : b) * s.length + tok) * (2 * D) + 2 * c;
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(f + i) = __ldg(reinterpret_cast<const float4*>(fr + i));
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int h = h0 + i * HPS;
    const bool live = h < s.heads;
    float e[8];
    float sum = 0.0f;
    if (live) {
      const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = Elem16<T>::unpack(u[j]);
        e[2 * j] = a.x;
        e[2 * j + 1] = a.y;
        sum = fmaf(a.x, a.x, fmaf(a.y, a.y, sum));
      }
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!live) continue;
    const float r = rsqrtf(sum * (1.0f / D) + s.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = e[j] * r * (w[j] + 1.0f);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = e[2 * j], z = e[2 * j + 1];
      if (s.freqs) {
        const float a1 = fmaf(f[4 * j], a, f[4 * j + 1] * z), z1 = fmaf(f[4 * j + 2], a, f[4 * j + 3] * z);
        a = a1;
        z = z1;
      }
      o[j] = Elem16<T>::pack(a, z);
    }
    T* y = static_cast<T*>(s.y) + (row * s.heads + h) * D + c;
    *reinterpret_cast<uint4*>(y) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace k2b
