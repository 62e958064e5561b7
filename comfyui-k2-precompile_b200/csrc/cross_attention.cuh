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
// which the matrix product asks for.  That costs up to 2^-8 (bf16) or 2^-11
// (fp16) of each probability, as much as the rounding of the output; an fp16 P
// below 2^-14 is off by up to 2^-25 instead (P is relative to the row's running
// maximum, or on the tile kernel to a reference up to 2^8 below it).  Row sums
// are taken of P before the rounding.
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
//
// Bound by latency: a warp's turn of 16 keys is one trip to memory, products
// and a join.  Measured: 1 query of 48/12 heads by 4096 keys (25 MB) 11.8 us;
// 16 queries of 20 heads of 64 by 729 keys, four latents, 9.6.
constexpr int XF_THREADS = 256;
constexpr int XF_WARPS = XF_THREADS / 32;
constexpr int XF_ROWS = 16;
constexpr int XF_KEYS = 16;
constexpr int XF_SPLITS = 8;  // CTAs of a cluster at most

template <int D>
constexpr int xf_smem_bytes() {
  return (XF_WARPS * XF_ROWS * D + XF_ROWS * D + 2 * XF_WARPS * XF_ROWS + 2 * XF_ROWS) * 4;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// CTAs per SM: two at D = 64 (within 128 registers), one at D = 128 (219).
__host__ __device__ constexpr int xf_per_sm(int dim) { return dim == 64 ? 2 : 1; }

template <typename T, int D>
__global__ void __launch_bounds__(XF_THREADS, D == 64 ? xf_per_sm(64) : 0) cross_few_kernel(const __grid_constant__ CrossParams p) {
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
    // V of keys 2t, 2t + 1, 2t + 8, 2t + 9; columns 64 e + 8 r..  (Loaded an
    // iteration earlier, behind the PV of the last, it measured slower: one
    // query by 4096 keys of 12 heads 17.0 against 13.8 us.)
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
  // four columns of a row to its place, rounded once
  auto store4 = [&](int at, float4 v, float sum) {
    const long long rr = (long long)rt * XF_ROWS + at / D;
    if (rr >= rows) return;
    const long long tok = rr / p.group, head = hk * p.group + rr % p.group;
    const float by = 1.0f / sum;
    uint2 o = make_uint2(0u, 0u);  // a row without keys
    if (sum != 0.0f) o = make_uint2(Elem16<T>::pack(v.x * by, v.y * by), Elem16<T>::pack(v.z * by, v.w * by));
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + ((long long)b * p.lq + tok) * p.heads * D + head * D + at % D) = o;
  };
  for (int at = 4 * threadIdx.x; at < XF_ROWS * D; at += 4 * XF_THREADS) {
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < XF_WARPS; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(so + w * XF_ROWS * D + at);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (p.splits == 1) {
      store4(at, sum, sml[XF_ROWS + at / D]);
    } else {
      *reinterpret_cast<float4*>(sred + at) = sum;
    }
  }
  if (p.splits == 1) return;
  // ---------------------------------------- join the CTAs of the cluster
  cluster_sync_all();
  const int share = XF_ROWS * D / p.splits;
  for (int i = 4 * threadIdx.x; i < share; i += 4 * XF_THREADS) {
    const int at = split * share + i, row = at / D;
    // everything in flight before the first is used
    float mc[XF_SPLITS], lc[XF_SPLITS];
    float4 vc[XF_SPLITS];
#pragma unroll
    for (int c = 0; c < XF_SPLITS; ++c) {
      mc[c] = -INFINITY, lc[c] = 0.0f;
      vc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c < p.splits) {
        mc[c] = ld_cluster_f32(cluster_map(smem_u32(sml + row), c));
        lc[c] = ld_cluster_f32(cluster_map(smem_u32(sml + XF_ROWS + row), c));
        vc[c] = ld_cluster_f32x4(cluster_map(smem_u32(sred + at), c));
      }
    }
    float top = -INFINITY, sum = 0.0f;
    float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < XF_SPLITS; ++c) top = fmaxf(top, mc[c]);
#pragma unroll
    for (int c = 0; c < XF_SPLITS; ++c) {
      const float f = mc[c] == -INFINITY ? 0.0f : exp2_fast((mc[c] - top) * kLog2e);
      sum = fmaf(lc[c], f, sum);
      val.x = fmaf(vc[c].x, f, val.x), val.y = fmaf(vc[c].y, f, val.y);
      val.z = fmaf(vc[c].z, f, val.z), val.w = fmaf(vc[c].w, f, val.w);
    }
    store4(at, val, sum);
  }
  cluster_sync_all();  // the others may still be reading this CTA's sums
}

// ------------------------------------------------------ tiles of queries
// Flash attention on tcgen05 for the many-query shapes.  One persistent CTA
// per SM walks a contiguous range of items; an item is two slots of 128
// queries that read the same KV head: two heads of an even GQA group at one
// token tile, or two token tiles of one head (odd groups).  Each K/V tile of
// 128 keys feeds both slots.
//
// TMEM (512 columns): S0 | S1 | O0 | O1 of 128 columns each; P (16-bit)
// overwrites the first 64 columns of its S.  Products issued by one thread
// execute in order, so S of the next tile may overwrite P behind the PV
// product that reads it, and S(j) being complete implies PV(j - 1) is.
//
// Warps: 0 the walk and its TMA loads, 1 and 3 products of slot 0 and 1, 2
// per-tile side data, 4-7 and 8-11 softmax and output of slot 0 and 1 (a
// thread owns a row).
//   - Warp 0 alone decides what is next: it writes one record per step (item,
//     key tile, ring slot, what to load and free) into a ring that the other
//     roles read, so that no division, length or mask lookup stands between a
//     barrier and the product behind it.
//   - A slot's products are issued by a warp of its own, as a whole warp with
//     one elected lane: descriptors are then in uniform registers (issued from
//     a one-lane branch, each product cost 80-100 cycles of scalar work against
//     64 of tensor time).  PV of a tile and S of the next go out together once
//     P is there; everything else they need was waited for before.
//   - Loads run ahead across items.  While a run of items has the same (b, KV
//     head) and all its tiles fit the ring, K and V stay where they are: a
//     short prompt is read once per CTA, not once per query tile.
//   - Warp 2 turns lengths, bias and key mask into a 128-bit word and 128
//     addends (log2 units) per tile, and zeroes the V rows of excluded keys
//     before the product may read them.  A tile with nothing to add and
//     nothing to exclude takes the path without either.
//   - A mask that depends on the query or the head is packed to bits by
//     cross_mask_kernel first (a row then reads 16 bytes per tile instead of
//     128, and all heads share them); tiles that no row of the item sees are
//     skipped by every role.
//   - O is rescaled in TMEM only when a row's maximum grew by more than 2^8
//     (P and the sum then stay within fp16 and fp32; o = O / l is the same).
//
// Bound by the chain S -> softmax -> PV of a slot (3700 cycles for 128 keys of
// both slots, 2050 of them products) and, for short prompts, by what an item
// costs at its end.  Measured: 8 x 4224 queries by 2048 keys, 48/12 heads, 1.65
// ms, 1030 TFLOP/s (1.84 ms, 925, once the power limit has lowered the clock);
// 4096 queries by 1000 keys under a regional mask 103 us; 2 x 4050 queries by 154
// and 76 keys with addends 88 us (200 MB).  Part of the exponentials as a
// polynomial on the FMA pipe measured slower.  The code's layout alone is worth
// 5%: compare builds, not edits.
constexpr int XT_BM = 128;
constexpr int XT_BN = 128;
constexpr int XT_THREADS = 384;
constexpr int XT_LAUNCH_REGS = 168;  // 65536 / 384; split 88 / 208 by setmaxnreg (128 x 88 + 256 x 208 = 384 x 168)
constexpr float XT_RESCALE = 8.0f;   // log2 units
// A row's reference is its maximum S * c, rounded: off by up to 2^-25 of it,
// which P carries as a power of two.  Up to 2^24 that is half a unit; from 2^28
// on P would leave fp16, from 2^32 on fp32.  A row with a larger maximum is done
// again by cross_row.
constexpr float XT_LARGEST = 16777216.0f;
constexpr int XT_RECORDS = 8;        // steps the walk may be ahead of the slowest role
constexpr int XT_READERS = 11;       // products (2), side data, eight softmax warps

template <int D>
struct XtShape {
  static constexpr int TILE = 128 * D * 2;            // bytes of a Q, K or V tile
  static constexpr int STAGES = D == 128 ? 2 : 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE;
  static constexpr int OFF_V = OFF_K + STAGES * TILE;
  static constexpr int OFF_O = OFF_V + STAGES * TILE;  // 4 KB per softmax warp
  static constexpr int OFF_AUX = OFF_O + 8 * 4096;
  static constexpr int AUX = 128 * 4 + 32;             // addends, keep words, flags
  static constexpr int OFF_REC = OFF_AUX + STAGES * AUX;
  static constexpr int OFF_BAR = OFF_REC + XT_RECORDS * 32;
  static constexpr int NBARS = 4 + 5 * STAGES + 8 + 2 * XT_RECORDS;
  static constexpr int SMEM = OFF_BAR + NBARS * 8 + 32 + 1024;
};

struct CrossMaps {
  CUtensorMap q, k, v;
};

struct CrossTileParams {
  CrossParams p;
  int pairs;            // slot pairs per KV head and token tile
  int qtiles;           // token tiles (of 128, or 256 where the slots are tiles)
  int qpair;            // slots are two token tiles of one head
  int nkt;              // key tiles of lk
  // packed mask (cross_mask_kernel) or null; row and column words by tile
  const uint4* bits;    // [mb, mh, mq, nkt]
  const uint4* cols;    // [mb, mh, ceil(mq / 128), nkt]: keys that some row of 128 sees
  int mb, mh, mq;       // extents of the packed mask (1 where broadcast)
};

// Packs a mask that depends on the query or the head: one CTA per 128 rows
// and 128 keys.
__global__ void __launch_bounds__(256)
    cross_mask_kernel(const uint8_t* mask, long long m_sb, long long m_sh, long long m_sq, long long m_sk, int planes,
                      int mh, int mq, int lk, int nkt, uint4* bits, uint4* cols) {
  pdl_launch_dependents();
  __shared__ uint32_t any[8][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kt = blockIdx.x % nkt, qt = blockIdx.x / nkt;
  const int plane = blockIdx.z * gridDim.y + blockIdx.y;  // of 65535 and more
  if (plane >= planes) return;
  const int b = plane / mh, h = plane % mh;
  uint32_t seen[4] = {0, 0, 0, 0};
  const uint8_t* base = mask + b * m_sb + h * m_sh;
  const int key0 = kt * 128 + lane;
  for (int i0 = 0; i0 < 16; i0 += 4) {  // 16 rows per warp, the loads of four in flight
    bool on[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = qt * 128 + warp * 16 + i0 + i;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int key = key0 + 32 * c;
        on[i][c] = row < mq && key < lk && __ldg(base + row * m_sq + key * m_sk) != 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = qt * 128 + warp * 16 + i0 + i;
      uint32_t w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        w[c] = __ballot_sync(0xffffffffu, on[i][c]);
        seen[c] |= w[c];
      }
      if (lane == 0 && row < mq)
        bits[((long long)plane * mq + row) * nkt + kt] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (lane < 4) any[warp][lane] = lane == 0 ? seen[0] : lane == 1 ? seen[1] : lane == 2 ? seen[2] : seen[3];
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t a[4] = {0, 0, 0, 0};
    for (int w = 0; w < 8; ++w)
      for (int c = 0; c < 4; ++c) a[c] |= any[w][c];
    cols[((long long)plane * ((mq + 127) / 128) + qt) * nkt + kt] = make_uint4(a[0], a[1], a[2], a[3]);
  }
}

// One step of the walk: key tile j of an item, or an item without any.
enum CrossFlags : int {
  XS_FIRST = 1,     // first tile of its item
  XS_LAST = 2,      // last tile of its item (also set for an item without tiles)
  XS_EMPTY = 4,     // no key: the output is zero and nothing else happens
  XS_LOAD = 8,      // K and V are loaded for this step (else they are still there)
  XS_FREE = 16,     // the ring slot is free after this step
  XS_END = 32,
};
struct CrossStep {
  // flags above, and for the products: ring slot << 8, its phase << 12, the
  // phase of the item's queries << 13
  int flags;
  int j, load, item_no;  // load: running number of the K/V load (ring slot load % STAGES)
  int b, hk, h0, q0;     // slot t: head h0 + t * hstep, tokens q0 + t * qstep..
};

// The keys of tile j that some row of the item sees (packed mask only).
__device__ __forceinline__ uint4 cross_seen(const CrossTileParams& P, int b, int h0, int q0, int j) {
  uint4 r = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int h = P.mh == 1 ? 0 : h0 + (P.qpair ? 0 : t);
    const int q = P.mq == 1 ? 0 : q0 + (P.qpair ? t * XT_BM : 0);
    if (q >= P.mq) continue;
    const long long row = ((long long)(P.mb == 1 ? 0 : b) * P.mh + h) * ((P.mq + 127) / 128) + q / 128;
    const uint4 c = P.cols[row * P.nkt + j];
    r.x |= c.x, r.y |= c.y, r.z |= c.z, r.w |= c.w;
  }
  return r;
}

// An addend in log2 units.  Past 2^127 those leave fp32: the rest of the range is
// laid out evenly over what fp32 has left, so that a finite addend stays finite
// and the larger of two stays the larger (one ulp there is 2^104: which of two
// keys gets all of the weight is all that an addend of this size says).
__device__ __forceinline__ float cross_addend(float raw) {
  constexpr float kPower = 1.7014118346046923e38f;  // 2^127
  const float size = fabsf(raw), low = fminf(size, kPower);
  return copysignf(fmaf(size - low, 0.55f, low * kLog2e), raw);
}

__device__ __forceinline__ int cross_keys(const CrossParams& p, int b) {
  return p.lengths ? min(max(__ldg(p.lengths + b), 0), p.lk) : p.lk;
}

// This CTA's items [range[0], range[1]): contiguous ranges of equal cost, an
// item costing its key tiles plus about two for its queries and output.
// (More than 64 latents: equal counts.)
__device__ __forceinline__ void cross_range(const CrossTileParams& P, int (&range)[2]) {
  const CrossParams& p = P.p;
  const int per = P.pairs * P.qtiles * p.kvheads;
  const int total = per * p.batch;
  if (!p.lengths || p.batch > 64) {
    range[0] = (int)((long long)total * blockIdx.x / gridDim.x);
    range[1] = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
    return;
  }
  long long all = 0;
  for (int b = 0; b < p.batch; ++b) all += (long long)per * ((cross_keys(p, b) + XT_BN - 1) / XT_BN + 2);
  const long long at[2] = {all * blockIdx.x / gridDim.x, all * (blockIdx.x + 1) / gridDim.x};
  long long before = 0;
  range[0] = range[1] = total;
  int e = 0;
  for (int b = 0; b < p.batch && e < 2; ++b) {
    const int cost = (cross_keys(p, b) + XT_BN - 1) / XT_BN + 2;
    while (e < 2 && at[e] < before + (long long)per * cost) {
      range[e] = b * per + (int)((at[e] - before) / cost);
      ++e;
    }
    before += (long long)per * cost;
  }
}

__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes;
}
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, "
      "rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// The larger of the two or three, NaN if any is.
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 128 columns of this lane's row, complete on return.
__device__ __forceinline__ void tmem_ld_row(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, "
      "%34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, "
      "%54, %55, %56, %57, %58, %59, %60, %61, %62, %63, %64, %65, %66, %67, %68, %69, %70, %71, %72, %73, "
      "%74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, "
      "%94, %95, %96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, "
      "%112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]),
        "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]),
        "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]),
        "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]),
        "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]),
        "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]),
        "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]),
        "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]),
        "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr)
      : "memory");
}
// 64 columns of this lane's row, complete on return.
__device__ __forceinline__ void tmem_ld_row(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, "
      "%34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, "
      "%54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_row(uint32_t taddr, const uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x64.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, "
      "%34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, "
      "%54, %55, %56, %57, %58, %59, %60, %61, %62, %63, %64};"
      ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(r[32]), "r"(r[33]), "r"(r[34]), "r"(r[35]),
        "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]), "r"(r[40]), "r"(r[41]), "r"(r[42]), "r"(r[43]), "r"(r[44]),
        "r"(r[45]), "r"(r[46]), "r"(r[47]), "r"(r[48]), "r"(r[49]), "r"(r[50]), "r"(r[51]), "r"(r[52]), "r"(r[53]),
        "r"(r[54]), "r"(r[55]), "r"(r[56]), "r"(r[57]), "r"(r[58]), "r"(r[59]), "r"(r[60]), "r"(r[61]), "r"(r[62]),
        "r"(r[63])
      : "memory");
}
__device__ __forceinline__ void tmem_st_row(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// One query's row by a warp on the FMA units, scores in natural units, so that
// the largest has an exponent of exactly 0 whatever its size (XT_LARGEST).  32
// keys at a time: a lane's own key for the score, its own columns for PV.  Out of
// line and once per item: a test of every tile's maximum, with S replaced by its
// rounded product, took 2 x 4050 queries by 154 keys from 87 to 90 us and 4096 by
// 1000 under a regional mask from 105 to 110.  1024 queries of 48/12 heads by 4096
// keys, every row done again: 22.9 ms, 0.15 without.  (165 cycles a key and row: the
// other roles' bounded waits last for a warp's 32 rows up to 700,000 keys.)
template <typename T, int D>
__device__ __noinline__ void cross_row(const CrossParams& p, int b, int head, int tok) {
  constexpr int C = D / 32;
  const int lane = threadIdx.x & 31, hk = head / p.group, n = cross_keys(p, b);
  const T* q = static_cast<const T*>(p.q) + b * p.q_sb + head * p.q_sh + tok * p.q_st;
  const T* k = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* v = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh + C * lane;
  float m = -INFINITY, l = 0.0f, o[C] = {};
  for (int k0 = 0; k0 < n; k0 += 32) {
    const int key = k0 + lane;
    bool keep = key < n;
    float s = 0.0f;
    if (keep && p.bias) {
      s = __ldg(p.bias + b * p.bias_sb + key);
      keep = s != -INFINITY;
    }
    if (keep && p.mask) keep = __ldg(p.mask + b * p.m_sb + head * p.m_sh + tok * p.m_sq + key * p.m_sk) != 0;
    if (keep) {
      const uint4* qr = reinterpret_cast<const uint4*>(q);
      const uint4* kr = reinterpret_cast<const uint4*>(k + key * p.k_st);
      float dot = 0.0f;
#pragma unroll 8
      for (int i = 0; i < D / 8; ++i) {
        const uint4 x = __ldg(qr + i), y = __ldg(kr + i);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 xf = Elem16<T>::unpack(xs[e]), yf = Elem16<T>::unpack(ys[e]);
          dot = fmaf(xf.x, yf.x, fmaf(xf.y, yf.y, dot));
        }
      }
      s = fmaf(dot, p.scale, s);
    } else {
      s = -INFINITY;
    }
    float next = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, w));
    next = fmaxf(next, m);
    const float f = m == -INFINITY ? 0.0f : exp2_fast((m - next) * kLog2e);
    const float e = keep ? exp2_fast((s - (next == -INFINITY ? 0.0f : next)) * kLog2e) : 0.0f;
    m = next;
    l = fmaf(l, f, e);
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] *= f;
    // (at scores of this size few weights are not 0)
    for (uint32_t live = __ballot_sync(0xffffffffu, e != 0.0f); live; live &= live - 1) {
      const int j = __ffs(live) - 1;
      const float pj = __shfl_sync(0xffffffffu, e, j);
      const uint32_t* vr = reinterpret_cast<const uint32_t*>(v + (k0 + j) * p.v_st);
#pragma unroll
      for (int i = 0; i < C; i += 2) {
        const float2 x = Elem16<T>::unpack(__ldg(vr + i / 2));
        o[i] = fmaf(pj, x.x, o[i]);
        o[i + 1] = fmaf(pj, x.y, o[i + 1]);
      }
    }
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  const float by = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (((long long)b * p.lq + tok) * p.heads + head) * D + C * lane);
#pragma unroll
  for (int i = 0; i < C; i += 2) dst[i / 2] = Elem16<T>::pack(o[i] * by, o[i + 1] * by);
}

template <typename T, int D>
__global__ void __launch_bounds__(XT_THREADS, 1)
    cross_tile_kernel(const __grid_constant__ CrossMaps maps, const __grid_constant__ CrossTileParams P) {
  using X = XtShape<D>;
  constexpr int NS = X::STAGES;
  constexpr int HALVES = D / 64;
  constexpr int BOX = 128 * 128;  // bytes of a 64-column half tile
  constexpr bool F16 = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + X::OFF_BAR);
  uint64_t* q_full = bars;               // [2]
  uint64_t* q_empty = q_full + 2;        // [2]
  uint64_t* k_full = q_empty + 2;        // [NS]
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* aux_full = v_empty + NS;
  uint64_t* s_full = aux_full + NS;      // [2]
  uint64_t* p_full = s_full + 2;         // [2]
  uint64_t* o_full = p_full + 2;         // [2]
  uint64_t* rec_full = o_full + 2;       // [XT_RECORDS]
  uint64_t* rec_empty = rec_full + XT_RECORDS;
  uint64_t* drained = rec_empty + XT_RECORDS;  // [2] teardown after an abort
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + X::NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int4* records = reinterpret_cast<int4*>(smem + X::OFF_REC);  // two per step
  const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
  const CrossParams& p = P.p;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const bool leader = elect_lane() != 0;  // products are ordered only within one thread

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
      mbar_init(&aux_full[i], 1);
    }
    for (int i = 0; i < XT_RECORDS; ++i) {
      mbar_init(&rec_full[i], 1);
      mbar_init(&rec_empty[i], XT_READERS);
    }
    mbar_init(drained, 1);
    mbar_init(drained + 1, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (P.bits) pdl_wait();  // the packed mask
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int hstep = P.qpair ? 0 : 1, qstep = P.qpair ? XT_BM : 0;

  // Record `no` of the walk, by a whole warp, and whether there is one (ok:
  // the wait for it).  Its place is free for the walk once every reader has it
  // in registers.
  // (the softmax warps wait inline: a call would cost them their registers)
  auto rec_ready = [&](uint32_t no) {
    return mbar_wait_fast(smem_u32(&rec_full[no % XT_RECORDS]), (no / XT_RECORDS) & 1, abort_addr, ERR_WAIT_LOAD);
  };
  auto read_step = [&](uint32_t no, CrossStep& st, bool ok) {
    const uint32_t at = no % XT_RECORDS;
    if (!__all_sync(0xffffffffu, ok)) return false;
    const int4 u = records[2 * at], v = records[2 * at + 1];
    st.flags = u.x, st.j = u.y, st.load = u.z, st.item_no = u.w;
    st.b = v.x, st.hk = v.y, st.h0 = v.z, st.q0 = v.w;
    __syncwarp();
    if (lane == 0) mbar_arrive(&rec_empty[at]);
    return (st.flags & XS_END) == 0;
  };

  // what is in flight, for the teardown after an abort
  int k_loads = 0, v_loads = 0, q_loads[2] = {0, 0};
  // (each share of the registers is set inside its branch: after a join ptxas would allocate for the smaller one)
  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // --------------------------------------------- softmax and output
    const int t = (warp - 4) >> 2;
    const int w4 = warp & 3;
    const int r = 32 * w4 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * w4) << 16);
    const uint32_t s_at = lane_base + t * 128, o_at = lane_base + 256 + t * 128;
    const float c = p.scale * kLog2e;
    uint32_t step = 0, out_no = 0;
    float m_run = -INFINITY, l_run = 0.0f;
    float largest = 0.0f;  // of the row's tile maxima without addends, where finite
    CrossStep st;
    for (uint32_t no = 0;
         read_step(no, st, mbar_wait_s(smem_u32(&rec_full[no % XT_RECORDS]), (no / XT_RECORDS) & 1, abort_addr, ERR_WAIT_SOFTMAX));
         ++no) {
      const int tok = st.q0 + t * qstep + r, head = st.h0 + t * hstep;
      const bool first = st.flags & XS_FIRST;
      if (first) {
        m_run = -INFINITY;
        l_run = 0.0f;
        largest = 0.0f;
      }
      if (!(st.flags & XS_EMPTY)) {
        const int s = st.load % NS;
        uint4 mine = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (P.bits) {
          const long long row = ((long long)(P.mb == 1 ? 0 : st.b) * P.mh + (P.mh == 1 ? 0 : head)) * P.mq +
                                (P.mq == 1 ? 0 : min(tok, P.mq - 1));
          mine = P.bits[row * P.nkt + st.j];
        }
        if (!mbar_wait_s(smem_u32(&aux_full[s]), (st.load / NS) & 1, abort_addr, ERR_WAIT_SOFTMAX) ||
            !mbar_wait_s(smem_u32(&s_full[t]), step & 1, abort_addr, ERR_WAIT_SOFTMAX)) break;
        ++step;
        tc_fence_after();
        const uint8_t* aux = smem + X::OFF_AUX + s * X::AUX;
        {
          const uint4 kw = *reinterpret_cast<const uint4*>(aux + 512);
          mine.x &= kw.x, mine.y &= kw.y, mine.z &= kw.z, mine.w &= kw.w;
        }
        const bool adds = *reinterpret_cast<const int*>(aux + 528) != 0;
        // Scores in log2 units are S * cm.  With addends they replace S first, in
        // a rolled loop: unrolled it costs the main path registers, and a spill
        // here goes to L2 (shared memory leaves L1 next to nothing).
        float cm = c;
        if (__builtin_expect(adds, 0)) {
          cm = 1.0f;
#pragma unroll 1
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t u[64];
            tmem_ld_row(s_at + 64 * cc, u);
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              const float4 a = *reinterpret_cast<const float4*>(aux + 4 * (64 * cc + e));
              u[e] = __float_as_uint(fmaf(__uint_as_float(u[e]), c, a.x));
              u[e + 1] = __float_as_uint(fmaf(__uint_as_float(u[e + 1]), c, a.y));
              u[e + 2] = __float_as_uint(fmaf(__uint_as_float(u[e + 2]), c, a.z));
              u[e + 3] = __float_as_uint(fmaf(__uint_as_float(u[e + 3]), c, a.w));
            }
            tmem_st_row(s_at + 64 * cc, u);
          }
          tmem_wait_st();
        }
        uint32_t u[128];
        tmem_ld_row(s_at, u);
        if (__builtin_expect(__any_sync(0xffffffffu, (mine.x & mine.y & mine.z & mine.w) != ~0u), 0)) {
          const uint32_t mw[4] = {mine.x, mine.y, mine.z, mine.w};
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (!((mw[e >> 5] >> (e & 31)) & 1u)) u[e] = 0xff800000u;  // -inf
        }
        float m4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m4[k] = __uint_as_float(u[k]);
#pragma unroll
          for (int jj = 1; jj < 31; jj += 2)
            m4[k] = fmax3_nan(m4[k], __uint_as_float(u[k + 4 * jj]), __uint_as_float(u[k + 4 * jj + 4]));
          m4[k] = fmax_nan(m4[k], __uint_as_float(u[k + 124]));
        }
        const float mx = cm * fmax_nan(fmax_nan(m4[0], m4[1]), fmax_nan(m4[2], m4[3]));
        if (!adds && fabsf(mx) < INFINITY) largest = fmaxf(largest, fabsf(mx));
        // m_run is the reference of P in log2 units: -inf until the row has
        // seen a key, NaN once a score was NaN or +inf (then the row is NaN)
        float alpha = 1.0f;
        bool rescale = false;
        if (mx > m_run + XT_RESCALE || m_run == -INFINITY || mx != mx) {
          const float next = mx == INFINITY ? __int_as_float(0x7fc00000) : mx;
          rescale = m_run != -INFINITY;
          if (rescale) alpha = exp2_fast(m_run - next);
          m_run = next;
        }
        const float base = m_run == -INFINITY ? 0.0f : m_run;
        const float2 cm2 = make_float2(cm, cm), base2 = make_float2(-base, -base);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int at = 64 * cc + 2 * e;
            float2 x = ffma2(make_float2(__uint_as_float(u[at]), __uint_as_float(u[at + 1])), cm2, base2);
            x.x = exp2_fast(x.x);
            x.y = exp2_fast(x.y);
            sum[e & 1] = fadd2(sum[e & 1], x);
            pk[e] = Elem16<T>::pack(x.x, x.y);
          }
          tmem_st_row(s_at + 32 * cc, pk);
        }
        const float2 all = fadd2(sum[0], sum[1]);
        l_run = fmaf(l_run, alpha, all.x + all.y);
        // O is stable here: S(j) being complete means PV(j - 1) is
        if (!first && __any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t u[16];
            tmem_ld16(o_at + 16 * cc, u);
            tmem_wait_ld_regs(u);
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * alpha);
            tmem_st16(o_at + 16 * cc, u);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!(st.flags & XS_LAST)) continue;
      const bool any = !(st.flags & XS_EMPTY);
      if (any) {
        if (!mbar_wait_s(smem_u32(&o_full[t]), out_no & 1, abort_addr, ERR_WAIT_SOFTMAX)) break;
        ++out_no;
        tc_fence_after();
      }
      // a row that saw no key is zero (its sum is 0, never NaN)
      const bool empty = l_run == 0.0f;
      const float inv = 1.0f / l_run;
      // 64 columns at a time through 4 KB of the warp's own, so that a store
      // writes four whole 128-byte lines (straight from the rows each wrote 32
      // sectors of 32 lines, and the output took as long as the tile)
      uint8_t* stage = smem + X::OFF_O + (warp - 4) * 4096;
      T* dst = static_cast<T*>(p.out) + (((long long)st.b * p.lq + st.q0 + t * qstep + 32 * w4) * p.heads + head) * D;
      const int left = p.lq - (st.q0 + t * qstep + 32 * w4);  // rows of this warp that exist
#pragma unroll 1
      for (int cc = 0; cc < D / 64; ++cc) {
        uint32_t u[64];
        tmem_ld_row(o_at + 64 * cc, u);  // (of an item without keys: not used)
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[e] = empty ? 0u : Elem16<T>::pack(__uint_as_float(u[8 * x + 2 * e]) * inv, __uint_as_float(u[8 * x + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int row = 4 * x + (lane >> 3), chunk = lane & 7;
          const uint4 o = *reinterpret_cast<const uint4*>(stage + row * 128 + ((chunk ^ (row & 7)) << 4));
          if (row < left)
            *reinterpret_cast<uint4*>(dst + (long long)row * p.heads * D + 64 * cc + 8 * chunk) = o;
        }
        __syncwarp();
      }
      uint32_t again = __ballot_sync(0xffffffffu, largest > XT_LARGEST && lane < left);
      for (; __builtin_expect(again != 0, 0); again &= again - 1)
        cross_row<T, D>(p, st.b, head, st.q0 + t * qstep + 32 * w4 + __ffs(again) - 1);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // --------------------------------------------- the walk and its loads
      if (lane == 0) {
        int range[2];
        cross_range(P, range);
        const int per = P.pairs * P.qtiles;
        int load = 0, item_no = 0, run_base = 0;
        uint32_t no = 0;
        auto put = [&](const CrossStep& st) {
          const uint32_t at = no % XT_RECORDS;
          if (no >= XT_RECORDS && !mbar_wait_fast(smem_u32(&rec_empty[at]), ((no / XT_RECORDS) & 1) ^ 1, abort_addr, ERR_WAIT_LOAD)) return false;
          records[2 * at] = make_int4(st.flags | (st.load % NS) << 8 | ((st.load / NS) & 1) << 12 | (st.item_no & 1) << 13, st.j,
                                      st.load, st.item_no);
          records[2 * at + 1] = make_int4(st.b, st.hk, st.h0, st.q0);
          mbar_arrive(&rec_full[at]);
          ++no;
          return true;
        };
        // a bounded wait for a place that a load may overwrite
        auto free_for = [&](const uint64_t* bar, uint32_t parity) {
          return mbar_wait_fast(smem_u32(bar), parity, abort_addr, ERR_WAIT_LOAD);
        };
        // D / 64 boxes of 128 rows from row y of head z
        auto fetch_tile = [&](const CUtensorMap* map, uint64_t* full, uint8_t* dst, int y, int z, int w) {
          mbar_arrive_expect_tx(full, X::TILE);
#pragma unroll 1
          for (int h = 0; h < HALVES; ++h) tma_load_4d(dst + h * BOX, map, full, 64 * h, y, z, w);
        };
        // what step st loads: the item's queries with its first tile, its K and V
        auto loads_of = [&](const CrossStep& st) {
          const int s = st.load % NS, kb = p.k_sb == 0 ? 0 : st.b;
          const uint32_t ph = ((st.load / NS) & 1) ^ 1;
          if (st.flags & XS_LOAD) {
            if (st.load >= NS && !free_for(&k_empty[s], ph)) return false;
            fetch_tile(&maps.k, &k_full[s], smem + X::OFF_K + s * X::TILE, st.j * XT_BN, st.hk, kb);
            k_loads = st.load + 1;
          }
          if (st.flags & XS_FIRST) {
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
              if (st.item_no > 0 && !free_for(&q_empty[t], (st.item_no - 1) & 1)) return false;
              fetch_tile(&maps.q, &q_full[t], smem + X::OFF_Q + t * X::TILE, st.q0 + t * qstep, st.h0 + t * hstep, st.b);
              q_loads[t] = st.item_no + 1;
            }
          }
          if (st.flags & XS_LOAD) {
            if (st.load >= NS && !free_for(&v_empty[s], ph)) return false;
            fetch_tile(&maps.v, &v_full[s], smem + X::OFF_V + s * X::TILE, st.j * XT_BN, st.hk, kb);
            v_loads = st.load + 1;
          }
          return true;
        };
        bool ok = true;
        CrossStep st;
        for (int i = range[0]; i < range[1] && ok; ++i) {
          const int key = i / per, rem = i % per;
          const int pair = rem / P.qtiles, qt = rem % P.qtiles;
          st.b = key / p.kvheads;
          st.hk = key % p.kvheads;
          st.h0 = st.hk * p.group + (P.qpair ? pair : 2 * pair);
          st.q0 = qt * (P.qpair ? 2 * XT_BM : XT_BM);
          const int tiles = (cross_keys(p, st.b) + XT_BN - 1) / XT_BN;
          const bool run_first = i == range[0] || rem == 0, run_last = i == range[1] - 1 || rem == per - 1;
          // K and V of a run of items stay when all their tiles fit the ring
          // (not under a packed mask: which V rows are zeroed depends on the item)
          const bool resident = !P.bits && tiles <= NS;
          if (resident && run_first) run_base = load, load += tiles;
          auto next_tile = [&](int j) {
            if (P.bits)
              for (; j < tiles; ++j) {
                const uint4 w = cross_seen(P, st.b, st.h0, st.q0, j);
                if (w.x | w.y | w.z | w.w) break;
              }
            return j;
          };
          st.j = next_tile(0);
          st.item_no = item_no;
          if (st.j >= tiles) {
            st.flags = XS_FIRST | XS_LAST | XS_EMPTY;
            st.load = 0;
            ok = put(st);
            continue;
          }
          ++item_no;
          for (int j = st.j, first = 1; j < tiles && ok; first = 0) {
            const int after = next_tile(j + 1);
            st.j = j;
            st.load = resident ? run_base + j : load++;
            st.flags = (first ? XS_FIRST : 0) | (after >= tiles ? XS_LAST : 0) | (!resident || run_first ? XS_LOAD : 0) |
                       (!resident || run_last ? XS_FREE : 0);
            ok = put(st) && loads_of(st);
            j = after;
          }
        }
        st.flags = XS_END;
        if (ok) put(st);
      }
    } else if (warp != 2) {
      // ------------------------------------------- products of slot t
      const int t = warp >> 1;
      constexpr uint32_t fmt = F16 ? 0 : 1;
      constexpr uint32_t idesc_s = make_idesc(1, fmt, fmt, 0, 0, XT_BM, XT_BN);  // Q K^T, both K-major
      constexpr uint32_t idesc_o = make_idesc(1, fmt, fmt, 0, 1, XT_BM, D);      // P V, V MN-major
      const uint32_t base = warp_uniform(smem_u32(smem));
      const uint32_t tm = warp_uniform(tmem);
      auto wait = [&](const uint64_t* bar, uint32_t parity) {
        return mbar_wait_fast(smem_u32(bar), parity, abort_addr, ERR_WAIT_MMA);
      };
      const uint64_t q_desc = umma_desc_sw128(base + X::OFF_Q + t * X::TILE, 16, 1024);
      const uint64_t k_desc = umma_desc_sw128(base + X::OFF_K, 16, 1024);
      const uint64_t v_desc = umma_desc_sw128(base + X::OFF_V, BOX, 1024);
      // PV of step w: 16 keys further are 16 rows of 128 B, the two 64-column
      // halves BOX apart (LBO); descriptors count 16 B
      auto issue_o = [&](int w) {
        const int s = (w >> 8) & 15;
        const uint64_t va = v_desc + s * (X::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_bf16_ts(tm + 256 + t * 128, tm + t * 128 + kk * 8, va + kk * (2048 >> 4), idesc_o,
                      kk > 0 || !(w & XS_FIRST) ? 1u : 0u);
        if (w & XS_LAST) mma_commit(&o_full[t]);
        if (w & XS_FREE) mma_commit(&v_empty[s]);
      };
      // S of step w: 16 columns further are 32 B on within a 64-column half,
      // BOX on to the next
      auto issue_s = [&](int w) {
        const int s = (w >> 8) & 15;
        const uint64_t ka = k_desc + s * (X::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
          mma_bf16_ss(tm + t * 128, q_desc + off, ka + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        mma_commit(&s_full[t]);
        if (w & XS_LAST) mma_commit(&q_empty[t]);
        if (w & XS_FREE) mma_commit(&k_empty[s]);
      };
      uint32_t no = 0;
      // the first word of the next step
      auto fetch = [&]() {
        const uint32_t at = no % XT_RECORDS;
        int w = rec_ready(no) ? records[2 * at].x : XS_END;
        w = warp_uniform(w);
        if (lane == 0) mbar_arrive(&rec_empty[at]);
        ++no;
        return w;
      };
      // cur: the step whose P comes next (XS_END: none), nxt: the step behind it,
      // whose S does.  One without keys takes its turn with nothing to issue: to
      // look past it for one with keys would hold back cur's PV, for which the
      // softmax warps wait, and with them the records that are being looked for.
      int cur = XS_END, nxt = fetch();
      uint32_t step = 0;
      bool ok = true;
      auto k_ready = [&](int w) { return wait(&k_full[(w >> 8) & 15], (w >> 12) & 1); };
      while (((cur & nxt) & XS_END) == 0) {
        // S of the item's next tile goes out behind PV; the first of another
        // item waits for its queries, which must not hold PV back
        bool s_due = !(nxt & (XS_END | XS_EMPTY));
        if (!(cur & XS_END)) {  // the side data of a ring slot are ready after its V
          const bool both = s_due && !(nxt & XS_FIRST);
          ok = wait(&aux_full[(cur >> 8) & 15], (cur >> 12) & 1) && (!both || k_ready(nxt)) && wait(&p_full[t], step & 1);
          if (!__all_sync(0xffffffffu, ok)) break;
          ++step;
          tc_fence_after();
          if (leader) {
            issue_o(cur);
            if (both) issue_s(nxt);
          }
          __syncwarp();
          s_due = s_due && !both;
        }
        if (s_due) {
          ok = k_ready(nxt) && wait(&q_full[t], (nxt >> 13) & 1);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
          if (leader) issue_s(nxt);
          __syncwarp();
        }
        cur = nxt & XS_EMPTY ? XS_END : nxt;
        if (!(nxt & XS_END)) nxt = fetch();
      }
    } else {
      // ---------------------------------------- side data of every K/V load
      CrossStep st;
      for (uint32_t no = 0; read_step(no, st, rec_ready(no)); ++no) {
        if (!(st.flags & XS_LOAD)) continue;
        const int s = st.load % NS, n = cross_keys(p, st.b);
        const bool key_mask = p.mask && !P.bits;
        float add[4];
        uint32_t word[4];
        bool plain = true;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = st.j * XT_BN + 32 * c + lane;
          bool keep = key < n;
          add[c] = 0.0f;
          if (keep && p.bias) {
            const float raw = __ldg(p.bias + st.b * p.bias_sb + key);
            keep = raw != -INFINITY;
            add[c] = keep ? cross_addend(raw) : 0.0f;
          }
          if (keep && key_mask) keep = __ldg(p.mask + st.b * p.m_sb + key * p.m_sk) != 0;
          word[c] = __ballot_sync(0xffffffffu, keep);
          plain = plain && !__any_sync(0xffffffffu, add[c] != 0.0f);
        }
        uint4 live = make_uint4(word[0], word[1], word[2], word[3]);
        if (P.bits) {
          const uint4 seen = cross_seen(P, st.b, st.h0, st.q0, st.j);
          live.x &= seen.x, live.y &= seen.y, live.z &= seen.z, live.w &= seen.w;
        }
        // the previous user of the slot is done once V has been loaded over it
        if (!__all_sync(0xffffffffu, mbar_wait_fast(smem_u32(&v_full[s]), (st.load / NS) & 1, abort_addr, ERR_WAIT_LOAD))) break;
        uint8_t* aux = smem + X::OFF_AUX + s * X::AUX;
#pragma unroll
        for (int c = 0; c < 4; ++c) reinterpret_cast<float*>(aux)[32 * c + lane] = add[c];
        if (lane == 0) {
          *reinterpret_cast<uint4*>(aux + 512) = make_uint4(word[0], word[1], word[2], word[3]);
          *reinterpret_cast<int*>(aux + 528) = plain ? 0 : 1;
        }
        // V rows of keys that nobody sees
        if (~(live.x & live.y & live.z & live.w)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const uint32_t lw = c < 2 ? (c ? live.y : live.x) : (c == 2 ? live.z : live.w);
            uint8_t* row = smem + X::OFF_V + s * X::TILE + (32 * c + lane) * 128;
#pragma unroll 1
            for (int x = 0; x < 8 * HALVES && !((lw >> lane) & 1u); ++x)
              *reinterpret_cast<uint4*>(row + (x >> 3) * BOX + 16 * (x & 7)) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux_full[s]);
      }
    }
  }

  // ------------------------------------------------------------ teardown
  __syncwarp();
  if (*abort_flag) {
    if (warp == 0 && lane == 0) {
      for (int t = 0; t < 2; ++t)
        if (q_loads[t]) mbar_drain(&q_full[t], (q_loads[t] - 1) & 1);
      for (int x = max(0, k_loads - NS); x < k_loads; ++x) mbar_drain(&k_full[x % NS], (x / NS) & 1);
      for (int x = max(0, v_loads - NS); x < v_loads; ++x) mbar_drain(&v_full[x % NS], (x / NS) & 1);
    }
    if ((warp == 1 || warp == 3) && leader) {  // behind every product issued
      mma_commit(drained + (warp >> 1));
      mbar_drain(drained + (warp >> 1), 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace k2b
