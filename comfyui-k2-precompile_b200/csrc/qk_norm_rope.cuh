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
// 256 values at once; a warp's item is one token and QKN_HEADS heads.  The
// warps of a resident wave walk over the items, and a warp loads its next item
// before it works on the present one, so that loads are always in flight.  The
// items of a token are neighbours: its table entries come from L1 after the
// first, and w + 1 is folded into them once per item.
// Measured: 4050 tokens of 48 + 12 heads of 128 out of a joint projection of 72
// (133 MB) 22.5 us, 5.9 TB/s; queries of 8 x 4224 tokens (842 MB) 132 us,
// 6.4 TB/s.
#pragma once
#include "elem16.cuh"

namespace k2b {

// Heads per warp item, as many loads in flight as 128 registers carry: with 8
// (three CTAs of 80 registers) 4050 tokens of 60 heads took 27.9 us, with 12
// 22.5, with 4 (four CTAs) 30.
constexpr int QKN_HEADS = 12;
constexpr int QKN_THREADS = 256;

struct QkNormSide {
  const void* x;
  void* y;            // [B, L, heads, D] contiguous
  const float* w;     // [D], "w+1" form
  const float* freqs; // [fb, L, D/2, 2, 2] or null
  long long sb, sh, st;
  int length, heads, fb;
  float eps;
  int chunks;         // ceil(heads / QKN_HEADS)
  uint32_t items;     // batch * length * chunks
};
struct QkNormParams {
  QkNormSide side[2];
};

// The items first, first + stride, .. of one side, by one warp.  (A function of
// the side, called with each of the two parameters: picked by index, every use
// of a parameter became a load of its own.)
template <typename T, int D>
__device__ __forceinline__ void qk_norm_side(const QkNormSide& s, uint32_t at, uint32_t stride) {
  constexpr int LPH = D / 8;               // lanes per head
  constexpr int HPS = 32 / LPH;            // heads per step
  constexpr int STEPS = QKN_HEADS / HPS;
  const int lane = threadIdx.x & 31;
  const int c = (lane % LPH) * 8;          // this lane's first column
  if (at >= s.items) return;

  struct Item {
    int h0;
    uint32_t b, tok;
  };
  auto locate = [&](uint32_t i) {
    Item it;
    const uint32_t row = i / s.chunks;     // batch * length + token
    it.h0 = (int)(i - row * s.chunks) * QKN_HEADS + lane / LPH;
    it.b = row / s.length;
    it.tok = row - it.b * s.length;
    return it;
  };
  auto load = [&](const Item& it, uint4 (&v)[STEPS]) {
    const T* x = static_cast<const T*>(s.x) + it.b * s.sb + it.tok * s.st + it.h0 * s.sh + c;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (it.h0 + i * HPS < s.heads) v[i] = ldg_stream(x);
      x += HPS * s.sh;
    }
  };
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(w + i) = __ldg(reinterpret_cast<const float4*>(s.w + c + i));
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] += 1.0f;

  Item it = locate(at);
  uint4 v[STEPS];
  load(it, v);
  for (;;) {
    const uint32_t next = at + stride;
    const bool more = next < s.items && next > at;
    Item nit = it;
    uint4 nv[STEPS];
    if (more) {
      nit = locate(next);
      load(nit, nv);
    }
    T* y = static_cast<T*>(s.y) + (((long long)it.b * s.length + it.tok) * s.heads + it.h0) * D + c;
    auto work = [&](auto turn) {
      float f[16];  // f[4 j ..]: the pair's matrix with the norm weights of its columns
      if constexpr (decltype(turn)::value) {
        const float* fr = s.freqs + ((long long)(s.fb == 1 ? 0 : it.b) * s.length + it.tok) * (2 * D) + 2 * c;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 m = __ldg(reinterpret_cast<const float4*>(fr + i));
          f[i] = m.x * w[i / 2], f[i + 1] = m.y * w[i / 2 + 1], f[i + 2] = m.z * w[i / 2], f[i + 3] = m.w * w[i / 2 + 1];
        }
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const bool live = it.h0 + i * HPS < s.heads;
        float e[8];
        float sum = 0.0f;
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = Elem16<T>::unpack(u[j]);
          e[2 * j] = a.x;
          e[2 * j + 1] = a.y;
          sum = fmaf(a.x, a.x, fmaf(a.y, a.y, sum));
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = rsqrtf(sum * (1.0f / D) + s.eps);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = e[2 * j] * r, z = e[2 * j + 1] * r;
          if constexpr (decltype(turn)::value) {
            o[j] = Elem16<T>::pack(fmaf(f[4 * j], a, f[4 * j + 1] * z), fmaf(f[4 * j + 2], a, f[4 * j + 3] * z));
          } else {
            o[j] = Elem16<T>::pack(w[2 * j] * a, w[2 * j + 1] * z);
          }
        }
        if (live) __stcs(reinterpret_cast<uint4*>(y + i * HPS * D), make_uint4(o[0], o[1], o[2], o[3]));
      }
    };
    if (s.freqs) {
      work(std::true_type{});
    } else {
      work(std::false_type{});
    }
    if (!more) break;
    at = next;
    it = nit;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) v[i] = nv[i];
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  const uint32_t stride = gridDim.x * (QKN_THREADS / 32);
  const uint32_t at = blockIdx.x * (QKN_THREADS / 32) + (threadIdx.x >> 5);
  qk_norm_side<T, D>(p.side[0], at, stride);
  // the second side goes on with the warp after the first side's last
  const uint32_t used = p.side[0].items % stride;
  qk_norm_side<T, D>(p.side[1], at >= used ? at - used : at + stride - used, stride);
}

}  // namespace k2b
