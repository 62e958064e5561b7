// cross_attention.cuh -- attention of one sequence's queries to another
// sequence's keys and values (a prompt's or an image encoder's states):
//
//   o = softmax(q k^T scale + bias) v   over the keys that are not excluded,
//   o = 0 for a row that has none left.
//
// Excluded are the keys at or past lengths[b], those whose bias is -inf and
// those whose mask byte is 0 (any broadcast of [B, H, lq, lk]).  What K holds
// at an excluded key is never used; V's values there are replaced by zeros
// wherever the key is excluded for all rows of a tile, because 0 * inf is not
// 0 (so V has to be finite only at keys that a mask hides from some queries
// and shows to others).
//
// Scores, row maxima, row sums and O are fp32; P is rounded to the type of V,
// which the matrix product asks for: 2^-9 (bf16) or 2^-12 (fp16) of each
// probability, as much as the rounding of the output.
#pragma once
#include "elem16.cuh"

namespace k2b {

constexpr float kLog2e = 1.4426950408889634f;

struct CrossParams {
  const void *q, *k, *v;
  void* out;               // [B, lq, heads * D]
  const int* lengths;      // [B] or null
  const uint8_t* mask;     // bytes, 0 = excluded, or null
  const float* bias;       // [.., lk] or null
  int batch, heads, kvheads, group, lq, lk;
  long long q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // elements; k_sb = v_sb = 0: shared by the batch
  long long m_sb, m_sh, m_sq, m_sk, bias_sb;
  float scale;
  int row_tiles, splits;
};

// ---------------------------------------------------- few rows per KV head
// The queries of the heads that share a KV head are one set of rows
// (row = token * group + head), 16 to a CTA, so every key and value is read
// once for all of them.  The keys go around the warps of the CTA, and of the
// cluster's CTAs (splits), 16 at a time; each warp keeps its own running
// maximum, sum and O, which are joined in a fixed order at the end: through
// shared memory inside the CTA, through the cluster's shared memory between
// them.  Nothing is staged: a lane loads 16 bytes of K that are two k16 steps
// of its B operand, and 16 bytes of V that are its column of eight n8 tiles
// (the order of d inside a product is free), and pairs the V rows of two keys
// with byte permutes.
constexpr int XF_THREADS = 256;
constexpr int XF_WARPS = XF_THREADS / 32;
constexpr int XF_ROWS = 16;
constexpr int XF_KEYS = 16;

template <int D>
constexpr int xf_smem_bytes() {
  return (XF_WARPS * XF_ROWS * D + XF_ROWS * D + 2 * XF_WARPS * XF_ROWS + 2 * XF_ROWS) * 4;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, int D>
__global__ void __launch_bounds__(XF_THREADS) cross_few_kernel(const __grid_constant__ CrossParams p) {
  extern __shared__ float xf_smem[];
  float* so = xf_smem;                            // [warps][16][D]
  float* sred = so + XF_WARPS * XF_ROWS * D;      // [16][D]
  float* sm = sred + XF_ROWS * D;                 // [warps][16]
  float* sl = sm + XF_WARPS * XF_ROWS;            // [warps][16]
  float* sml = sl + XF_WARPS * XF_ROWS;           // [16] max, [16] sum of the CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits;
  const int rt = (blockIdx.x / p.splits) % p.row_tiles;
  const int bh = blockIdx.x / (p.splits * p.row_tiles);
  const int b = bh / p.kvheads, hk = bh % p.kvheads;
  const long long rows = (long long)p.group * p.lq;
  int n = p.lk;
  if (p.lengths) n = min(max(__ldg(p.lengths + b), 0), p.lk);

  // Q: rows r and r + 8 of the tile, columns 32 j + 8 t..
  uint4 qa[D / 32], qb[D / 32];
  const long long ra = (long long)rt * XF_ROWS + r, rb = ra + 8;
  const bool la = ra < rows, lb = rb < rows;
  {
    const T* q = static_cast<const T*>(p.q) + b * p.q_sb + 8 * t;
    const T* pa = q + (hk * p.group + (la ? ra % p.group : 0)) * p.q_sh + (la ? ra / p.group : 0) * p.q_st;
    const T* pb = q + (hk * p.group + (lb ? rb % p.group : 0)) * p.q_sh + (lb ? rb / p.group : 0) * p.q_st;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      qa[j] = __ldg(reinterpret_cast<const uint4*>(pa + 32 * j));
      qb[j] = __ldg(reinterpret_cast<const uint4*>(pb + 32 * j));
    }
  }
  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh + 8 * t;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh + 8 * r;
  const uint8_t *mrow_a = nullptr, *mrow_b = nullptr;
  if (p.mask) {
    mrow_a = p.mask + b * p.m_sb + (hk * p.group + (la ? ra % p.group : 0)) * p.m_sh + (la ? ra / p.group : 0) * p.m_sq;
    mrow_b = p.mask + b * p.m_sb + (hk * p.group + (lb ? rb % p.group : 0)) * p.m_sh + (lb ? rb / p.group : 0) * p.m_sq;
  }
  const float* bias = p.bias ? p.bias + b * p.bias_sb : nullptr;

  float o[D / 64][8][4];
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[e][j][c] = 0.0f;
  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;

  const int tiles = (n + XF_KEYS - 1) / XF_KEYS;
  const int stride = p.splits * XF_WARPS;
  uint4 kf[2][D / 32];
  auto load_k = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const T* kp = kbase + (long long)min(tile * XF_KEYS + 8 * i + r, n - 1) * p.k_st;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) kf[i][j] = ldg_stream(kp + 32 * j);
    }
  };
  int tile = split * XF_WARPS + warp;
  if (tile < tiles) load_k(tile);
  for (; tile < tiles; tile += stride) {
    const int k0 = tile * XF_KEYS;
    // V of keys 2t, 2t + 1, 2t + 8, 2t + 9; columns 64 e + 8 r..
    uint4 vf[4][D / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* vp = vbase + (long long)min(k0 + 2 * t + (i & 1) + 8 * (i >> 1), n - 1) * p.v_st;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) vf[i][e] = ldg_stream(vp + 64 * e);
    }
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        mma16816<T>(s[i], qa[j].x, qb[j].x, qa[j].y, qb[j].y, kf[i][j].x, kf[i][j].y);
        mma16816<T>(s[i], qa[j].z, qb[j].z, qa[j].w, qb[j].w, kf[i][j].z, kf[i][j].w);
      }
    }
    if (tile + stride < tiles) load_k(tile + stride);
    // scores in natural units; keep[i][c]: key 2t + c + 8i for rows r (bit 0) and r + 8 (bit 1)
    bool dead[4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int key = k0 + 8 * i + 2 * t + c;
        bool ka = key < n, kb = ka;
        float add = 0.0f;
        if (ka && bias) {
          add = __ldg(bias + key);
          ka = kb = add != -INFINITY;
        }
        if (ka && p.mask) {
          ka = __ldg(mrow_a + key * p.m_sk) != 0;
          kb = __ldg(mrow_b + key * p.m_sk) != 0;
        }
        s[i][c] = ka ? fmaf(s[i][c], p.scale, add) : -INFINITY;
        s[i][2 + c] = kb ? fmaf(s[i][2 + c], p.scale, add) : -INFINITY;
        dead[2 * i + c] = (__ballot_sync(0xffffffffu, (ka && la) || (kb && lb)) & (0x11111111u << t)) == 0;
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (dead[i]) {
#pragma unroll
        for (int e = 0; e < D / 64; ++e) vf[i][e] = make_uint4(0u, 0u, 0u, 0u);
      }
    float xa = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    float xb = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
      xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, w));
      xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, w));
    }
    if (__any_sync(0xffffffffu, xa > m_a || xb > m_b)) {
      const float na = fmaxf(m_a, xa), nb = fmaxf(m_b, xb);
      // a row without any key so far has m = -inf and nothing to rescale
      const float fa = m_a == -INFINITY ? 0.0f : exp2_fast((m_a - na) * kLog2e);
      const float fb = m_b == -INFINITY ? 0.0f : exp2_fast((m_b - nb) * kLog2e);
      m_a = na, m_b = nb;
      l_a *= fa, l_b *= fb;
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[e][j][0] *= fa, o[e][j][1] *= fa;
          o[e][j][2] *= fb, o[e][j][3] *= fb;
        }
    }
    const float base_a = m_a == -INFINITY ? 0.0f : m_a, base_b = m_b == -INFINITY ? 0.0f : m_b;
    uint32_t pf[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float p0 = exp2_fast((s[i][0] - base_a) * kLog2e), p1 = exp2_fast((s[i][1] - base_a) * kLog2e);
      const float p2 = exp2_fast((s[i][2] - base_b) * kLog2e), p3 = exp2_fast((s[i][3] - base_b) * kLog2e);
      l_a += p0 + p1;
      l_b += p2 + p3;
      pf[2 * i] = Elem16<T>::pack(p0, p1);
      pf[2 * i + 1] = Elem16<T>::pack(p2, p3);
    }
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const uint32_t v0[4] = {vf[0][e].x, vf[0][e].y, vf[0][e].z, vf[0][e].w};
      const uint32_t v1[4] = {vf[1][e].x, vf[1][e].y, vf[1][e].z, vf[1][e].w};
      const uint32_t v2[4] = {vf[2][e].x, vf[2][e].y, vf[2][e].z, vf[2][e].w};
      const uint32_t v3[4] = {vf[3][e].x, vf[3][e].y, vf[3][e].z, vf[3][e].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        mma16816<T>(o[e][j], pf[0], pf[1], pf[2], pf[3], __byte_perm(v0[j >> 1], v1[j >> 1], sel),
                    __byte_perm(v2[j >> 1], v3[j >> 1], sel));
      }
    }
  }

  // -------------------------------------------- join the warps of the CTA
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    l_a += __shfl_xor_sync(0xffffffffu, l_a, w);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, w);
  }
  if (t == 0) {
    sm[warp * XF_ROWS + r] = m_a;
    sm[warp * XF_ROWS + r + 8] = m_b;
    sl[warp * XF_ROWS + r] = l_a;
    sl[warp * XF_ROWS + r + 8] = l_b;
  }
  __syncthreads();
  float ta = -INFINITY, tb = -INFINITY;
#pragma unroll
  for (int w = 0; w < XF_WARPS; ++w) {
    ta = fmaxf(ta, sm[w * XF_ROWS + r]);
    tb = fmaxf(tb, sm[w * XF_ROWS + r + 8]);
  }
  const float fa = m_a == -INFINITY ? 0.0f : exp2_fast((m_a - ta) * kLog2e);
  const float fb = m_b == -INFINITY ? 0.0f : exp2_fast((m_b - tb) * kLog2e);
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        float* at = so + (warp * XF_ROWS + r) * D + 64 * e + 16 * t + 8 * c + j;
        *reinterpret_cast<float4*>(at) =
            make_float4(o[e][j][c] * fa, o[e][j + 1][c] * fa, o[e][j + 2][c] * fa, o[e][j + 3][c] * fa);
        *reinterpret_cast<float4*>(at + 8 * D) = make_float4(o[e][j][2 + c] * fb, o[e][j + 1][2 + c] * fb,
                                                             o[e][j + 2][2 + c] * fb, o[e][j + 3][2 + c] * fb);
      }
  if (threadIdx.x < XF_ROWS) {
    const int row = threadIdx.x;
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < XF_WARPS; ++w) top = fmaxf(top, sm[w * XF_ROWS + row]);
    for (int w = 0; w < XF_WARPS; ++w) {
      const float mw = sm[w * XF_ROWS + row];  // factor 0, not a skip: a sum of NaN scores stays NaN
      sum = fmaf(sl[w * XF_ROWS + row], mw == -INFINITY ? 0.0f : exp2_fast((mw - top) * kLog2e), sum);
    }
    sml[row] = top;
    sml[XF_ROWS + row] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < XF_ROWS * D; i += XF_THREADS) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < XF_WARPS; ++w) sum += so[w * XF_ROWS * D + i];
    sred[i] = sum;
  }
  // ---------------------------------------- join the CTAs of the cluster
  if (p.splits > 1) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  const int share = XF_ROWS * D / p.splits;
  for (int i = threadIdx.x; i < share; i += XF_THREADS) {
    const int at = split * share + i;
    const int row = at / D, d = at % D;
    const long long rr = (long long)rt * XF_ROWS + row;
    float top = -INFINITY, sum = 0.0f, val = 0.0f;
    if (p.splits == 1) {
      sum = sml[XF_ROWS + row];
      val = sred[at];
    } else {
      for (int c = 0; c < p.splits; ++c)
        top = fmaxf(top, ld_cluster_f32(cluster_map(smem_u32(sml + row), c)));
      for (int c = 0; c < p.splits; ++c) {
        const float mc = ld_cluster_f32(cluster_map(smem_u32(sml + row), c));
        const float f = mc == -INFINITY ? 0.0f : exp2_fast((mc - top) * kLog2e);
        sum = fmaf(ld_cluster_f32(cluster_map(smem_u32(sml + XF_ROWS + row), c)), f, sum);
        val = fmaf(ld_cluster_f32(cluster_map(smem_u32(sred + at), c)), f, val);
      }
    }
    if (rr < rows) {
      const long long tok = rr / p.group, head = hk * p.group + rr % p.group;
      static_cast<T*>(p.out)[((long long)b * p.lq + tok) * p.heads * D + head * D + d] =
          Elem16<T>::from_float(sum == 0.0f ? 0.0f : val / sum);
    }
  }
  if (p.splits > 1) cluster_sync_all();  // the others may still be reading this CTA's sums
}

}  // namespace k2b
