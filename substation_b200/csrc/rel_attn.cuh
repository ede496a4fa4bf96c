// Attention with a bias per head and relative position on tcgen05 (included by gemm.cu; shares its TMA / tcgen05 helpers).
//
//   out[p,j] = sum_k softmax_k(scale * q.k + bias[k - pos(j)]) v[p,k]
//
// The bias of a head is one row of floats over relative positions: bias_rows[head][rel + reach + kPad], written by
// expand_bias_kernel in units of log2, constant from `reach` on in both directions and continued kPad entries further, so that a
// tile which touches the varying part reads it without clamping.  A tile wholly outside has one bias.
//
// Projections are [rows x features] tiles with 128-byte swizzle, 64 features a box; heads of up to 64 features run as 64, up to
// 128 as 128 (the tensor map's bounds fill the rest with zeros).

#pragma once

namespace rel {

constexpr int kPad = 160;                            // 128 columns and the 32 rows of a warp
constexpr float kLazy = 8.f;                         // log2 units a row's reference may lag behind its maximum

struct Common {
  int J, K, H, G, B, P;
  float c2;                                          // scale * log2(e)
  int causal;
  const int* lengths;
  const int* first;
  const float* bias_rows;
  int pitch, reach;                                  // floats of a row; first distance of the last bucket
};

__device__ __forceinline__ int keys_of(const Common& c, int b) {
  return c.lengths ? max(0, min(c.K, __ldg(c.lengths + b))) : c.K;
}
__device__ __forceinline__ int first_of(const Common& c, int b) {
  return c.first ? max(-(1 << 29), min(1 << 29, __ldg(c.first + b))) : 0;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// D (+)= A * B with A in tensor memory (16-bit pairs, a row per lane)
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// ROWS rows x P features of one head and sample, from row r0 (rows and features beyond the tensor arrive as zeros)
template <int P, int ROWS>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int r0, int h, int b) {
#pragma unroll
  for (int x = 0; x < P / 64; ++x) tma_load_4d(dst + x * (ROWS * 128), map, bar, x * 64, r0, h, b);
}
// D[128 x N] = A rows [128 x P] times B rows [N x P], over the features
template <int P, int N>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b) {
  const uint32_t idesc = (1u << 4) | SB_IDESC_AB_FMT | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
  const uint64_t da = make_desc(a, 16u, 1024u), db = make_desc(b, 16u, 1024u);
#pragma unroll
  for (int k = 0; k < P / 16; ++k)
    umma_f16(d, da + (uint64_t)((k >> 2) * (128 * 8) + (k & 3) * 2), db + (uint64_t)((k >> 2) * (N * 8) + (k & 3) * 2), idesc,
             k > 0 ? 1u : 0u);
}
// D[128 x P] (+)= S[128 x K] * B, S in tensor memory and B [K rows x P features] in shared memory
template <int P, int K>
__device__ __forceinline__ void mma_weighted(uint32_t d, uint32_t s, uint32_t b, bool accumulate) {
  const uint32_t idesc = (1u << 4) | SB_IDESC_AB_FMT | (1u << 16) | ((uint32_t)(P >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
  const uint64_t db = make_desc(b, (uint32_t)(K * 128), 1024u);
#pragma unroll
  for (int k = 0; k < K / 16; ++k)
    umma_f16_ts(d, s + (uint32_t)(k * 8), db + (uint64_t)(k * 128), idesc, (accumulate || k > 0) ? 1u : 0u);
}
// Rows from `valid` on of a [ROWS x P] tile become zeros: 0 * what stands behind a sequence's end must be 0.
template <int P, int ROWS>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int valid, int lane) {
#pragma unroll
  for (int x = 0; x < P / 64; ++x)
    for (int i = valid * 8 + lane; i < ROWS * 8; i += 32) *reinterpret_cast<uint4*>(tile + x * (ROWS * 128) + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
// 32 accumulator columns -> alpha * value, 16-bit, the first n of them, at ptr[p * sP]
__device__ __forceinline__ void store_features(sb_half* ptr, long long sP, const uint32_t* r, float alpha, int n) {
  if (sP == 1 && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && (n & 7) == 0) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint4 o;
      uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = flash::pack2(__uint_as_float(r[v * 8 + 2 * e]) * alpha, __uint_as_float(r[v * 8 + 2 * e + 1]) * alpha);
      if (v * 8 < n) reinterpret_cast<uint4*>(ptr)[v] = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < n) ptr[e * sP] = sb_f2h(__uint_as_float(r[e]) * alpha);
  }
}

// ---- forward ---------------------------------------------------------------------------------------------------
constexpr int kFwdThreads = 192;                     // producer warp, MMA warp, four softmax warps

struct FwdParams {
  Common c;
  int nq, units, chunk;                              // query tiles of a unit; units = H * B; units taken together
  int items;
  Proj out;
  RelRows lse;
};

// The i-th work item: a tile of queries of one head and sample.  Units go in chunks, and within a chunk the last tiles first:
// with a causal span these are the long ones, and one head's keys stay in L2 while its tiles are worked on.
struct Item { int b, h, t, first, keys, tiles; };
__device__ __forceinline__ Item item_of(const FwdParams& p, int i) {
  Item it;
  const int per = p.chunk * p.nq, c = i / per, r = i % per;
  const int here = min(p.chunk, p.units - c * p.chunk), unit = c * p.chunk + r % here;
  it.t = p.nq - 1 - r / here;
  it.b = unit / p.c.H;
  it.h = unit % p.c.H;
  it.first = first_of(p.c, it.b);
  it.keys = keys_of(p.c, it.b);
  if (p.c.causal) it.keys = max(0, min(it.keys, it.first + min(p.c.J, it.t * 128 + 128)));
  it.tiles = (it.keys + 127) >> 7;
  return it;
}

// Shared memory of a CTA (two per SM): query tiles, the ring of key and value tiles, two rows of biases, barriers.
template <int P>
struct FwdCfg {
  static constexpr int kTile = 128 * P * 2;
  static constexpr int kQ = P == 64 ? 2 : 1;         // query tiles (the next item's is fetched early)
  static constexpr int kRing = P == 64 ? 4 : 2;
  static constexpr int kTiles = (kQ + kRing) * kTile;
  static constexpr bool kAlias = P == 128;           // the exponentials overwrite their scores
  static constexpr uint32_t kPm = kAlias ? 0 : 128, kO = kAlias ? 128 : 192;   // tensor memory columns; scores at 0
  static int smem(int pitch) { return kTiles + 2 * pitch * 4 + 1024 + 256; }
};

// One tile of scores of a thread's row against its 128 keys.  NEAR: the bias varies, bp[c] is column c's; else it is `flat`.
// MASK: columns from lim on are hidden.
template <bool NEAR, bool MASK>
__device__ __forceinline__ float row_max(uint32_t s, const float* bp, float flat, int lim, float c2) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t r[32];
    tmem_ld32_nowait(s + c * 32, r);
    float b[32];
    if (NEAR) {
#pragma unroll
      for (int e = 0; e < 32; ++e) b[e] = bp[c * 32 + e];
    }
    attn::tmem_ld_wait32(r);
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      float t = __uint_as_float(r[e]);
      if (NEAR) t = fmaf(t, c2, b[e]);
      if (MASK && c * 32 + e >= lim) t = -INFINITY;
      mx[e & 3] = fmaxf(mx[e & 3], t);
    }
  }
  const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  return NEAR || m == -INFINITY ? m : fmaf(m, c2, flat);
}
// Exponentials against 2^ref as 16-bit pairs into tensor memory; returns their sum.
template <bool NEAR, bool MASK>
__device__ __forceinline__ float row_exp(uint32_t s, uint32_t dst, const float* bp, float flat, float ref, int lim, float c2) {
  float l0 = 0.f, l1 = 0.f;
  const float off = flat - ref;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t r[32], w[16];
    tmem_ld32_nowait(s + c * 32, r);
    float b[32];
    if (NEAR) {
#pragma unroll
      for (int e = 0; e < 32; ++e) b[e] = bp[c * 32 + e] - ref;
    }
    attn::tmem_ld_wait32(r);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float x = fmaf(__uint_as_float(r[2 * e]), c2, NEAR ? b[2 * e] : off);
      float y = fmaf(__uint_as_float(r[2 * e + 1]), c2, NEAR ? b[2 * e + 1] : off);
      if (MASK) {
        if (c * 32 + 2 * e >= lim) x = -INFINITY;
        if (c * 32 + 2 * e + 1 >= lim) y = -INFINITY;
      }
      x = attn::ex2_approx(x);
      y = attn::ex2_approx(y);
      l0 += x;
      l1 += y;
      w[e] = flash::pack2(x, y);
    }
    tmem_st16(dst + c * 16, w);
  }
  return l0 + l1;
}

// One CTA: 128 queries of one unit against its keys in tiles of 128; two CTAs per SM, so that one's tensor and copy work runs
// beside the other's softmax.  Tensor memory: scores [128 x 128], their exponentials as 16-bit pairs (the second product's
// operand comes from there) and the output [128 x P].  Softmax warps: thread = row, exponentials against a reference that may
// lag 2^8 behind the maximum; only beyond is the output rescaled.
template <int P>
__global__ void __launch_bounds__(kFwdThreads, 2)
rel_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
               const __grid_constant__ FwdParams p) {
  using Cfg = FwdCfg<P>;
  constexpr int kRing = Cfg::kRing, kQ = Cfg::kQ;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sq = (raw + 1023u) & ~1023u, ring = sq + kQ * Cfg::kTile;
  const uint32_t sbias = sq + Cfg::kTiles, bars = sbias + 2u * p.c.pitch * 4u;
  const uint32_t q_full = bars, q_empty = bars + 16, s_full = bars + 32, p_full = bars + 40, p_free = bars + 48, o_empty = bars + 56;
  const uint32_t b_full = bars + 64, b_empty = bars + 80, kv_full = bars + 96, kv_empty = kv_full + 8 * kRing;
  uint8_t* gen = smem_raw + (sq - raw);
  const float* bias_s = reinterpret_cast<const float*>(gen + (sbias - sq));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + (kv_empty + 8 * kRing - sq));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_empty + 8 * i, 4);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 4);
    mbar_init(p_free, 1);
    mbar_init(o_empty, 4);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(kv_full + 8 * i, 1);
      mbar_init(kv_empty + 8 * i, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmQ) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  grid_dependency_sync();

  // `it` counts the items that see a key, n their key tiles
  if (warp == 0) {
    // ---------------- producer: queries and biases of the item, then its keys and values in turn ----------------
    uint32_t it = 0, x = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
      const Item w = item_of(p, item);
      if (w.tiles == 0) continue;
      const uint32_t qb = it % kQ, bb = it & 1u;
      ok = __all_sync(0xffffffffu, mbar_wait(q_empty + 8 * qb, ((it / kQ) & 1u) ^ 1u, 41)) &&
           __all_sync(0xffffffffu, mbar_wait(b_empty + 8 * bb, ((it >> 1) & 1u) ^ 1u, 41));
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(q_full + 8 * qb, Cfg::kTile);
        load_rows<P, 128>(sq + qb * Cfg::kTile, &tmQ, q_full + 8 * qb, w.t * 128, w.h, w.b);
        mbar_expect_tx(b_full + 8 * bb, p.c.pitch * 4);
        bulk_load(sbias + bb * p.c.pitch * 4, p.c.bias_rows + (long long)w.h * p.c.pitch, p.c.pitch * 4, b_full + 8 * bb);
      }
      __syncwarp();
      const int hk = w.h / (p.c.H / p.c.G);
      for (int i = 0; i < 2 * w.tiles; ++i, ++x) {       // even: keys of tile i / 2, odd: its values
        const uint32_t s = x % kRing;
        ok = __all_sync(0xffffffffu, mbar_wait(kv_empty + 8 * s, ((x / kRing) & 1u) ^ 1u, 41));
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(kv_full + 8 * s, Cfg::kTile);
          load_rows<P, 128>(ring + s * Cfg::kTile, i & 1 ? &tmV : &tmK, kv_full + 8 * s, (i >> 1) * 128, hk, w.b);
        }
        __syncwarp();
      }
      ++it;
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    uint32_t it = 0, n = 0, x = 0;                       // x: ring uses before this item
    bool ok = true;
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
      const Item w = item_of(p, item);
      if (w.tiles == 0) continue;
      const uint32_t qb = it % kQ;
      auto slot_full = [&](uint32_t use) {
        ok = __all_sync(0xffffffffu, mbar_wait(kv_full + 8 * (use % kRing), (use / kRing) & 1u, 42));
        tc_fence_after();
        return ok;
      };
      auto scores = [&](int i) {
        const uint32_t use = x + 2u * i, s = use % kRing;
        if (!slot_full(use)) return;
        if (flash::elect_one()) {
          mma_rows<P, 128>(tmem, sq + qb * Cfg::kTile, ring + s * Cfg::kTile);
          umma_commit(s_full);
          umma_commit(kv_empty + 8 * s);
          if (i == w.tiles - 1) umma_commit(q_empty + 8 * qb);
        }
        __syncwarp();
      };
      ok = __all_sync(0xffffffffu, mbar_wait(q_full + 8 * qb, (it / kQ) & 1u, 42));
      if (!ok) break;
      scores(0);
      for (int i = 0; i < w.tiles && ok; ++i, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait(p_full, n & 1u, 43));   // the scores have been read, their exponentials written
        if (!ok) break;
        tc_fence_after();
        if (!Cfg::kAlias && i + 1 < w.tiles) scores(i + 1);
        if (!ok) break;
        const uint32_t use = x + 2u * i + 1u, s = use % kRing;
        if (!slot_full(use)) break;
        if (w.keys - i * 128 < 128) zero_rows<P, 128>(gen + (ring - sq) + s * Cfg::kTile, w.keys - i * 128, lane);
        if (i == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(o_empty, (it & 1u) ^ 1u, 44));
          if (!ok) break;
          tc_fence_after();
        }
        if (flash::elect_one()) {
          mma_weighted<P, 128>(tmem + Cfg::kO, tmem + Cfg::kPm, ring + s * Cfg::kTile, i > 0);
          umma_commit(kv_empty + 8 * s);
          umma_commit(p_free);
        }
        __syncwarp();
        if (Cfg::kAlias && i + 1 < w.tiles) scores(i + 1);
      }
      x += 2u * w.tiles;
      ++it;
    }
  } else {
    // ---------------- softmax warps: thread = one query ----------------
    const int q = warp & 3;
    const int rt = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t ts = tmem + lanes, tp = ts + Cfg::kPm, to = ts + Cfg::kO;
    uint32_t n = 0, it = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
      const Item w = item_of(p, item);
      const int j = w.t * 128 + rt, pos = w.first + j;
      const bool row = j < p.c.J;
      int mine = w.keys;                                 // keys that this row sees
      if (p.c.causal) mine = min(mine, pos + 1);
      float m = -INFINITY, l = 0.f;
      const uint32_t bb = it & 1u;
      const float* bias = bias_s + bb * p.c.pitch;
      if (w.tiles > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_full + 8 * bb, (it >> 1) & 1u, 45));
        if (!ok) break;
      }
      for (int kb = 0; kb < w.tiles; ++kb, ++n) {
        const int lim = mine - kb * 128;
        const int rel0 = kb * 128 - pos;                 // relative position of the first column
        const int lo = kb * 128 - (w.first + w.t * 128 + q * 32 + 31), hi = kb * 128 + 127 - (w.first + w.t * 128 + q * 32);
        const bool near = hi > -p.c.reach && lo < p.c.reach;
        const float flat = near ? 0.f : bias[kPad + (lo >= p.c.reach ? 2 * p.c.reach : 0)];
        const float* bp = bias + (near ? rel0 + p.c.reach + kPad : 0);
        const bool mask = __any_sync(0xffffffffu, lim < 128);
        ok = __all_sync(0xffffffffu, mbar_wait(s_full, n & 1u, 46));
        if (!ok) break;
        tc_fence_after();
        float mx;
        if (near) mx = mask ? row_max<true, true>(ts, bp, 0.f, lim, p.c.c2) : row_max<true, false>(ts, bp, 0.f, lim, p.c.c2);
        else mx = mask ? row_max<false, true>(ts, bp, flat, lim, p.c.c2) : row_max<false, false>(ts, bp, flat, lim, p.c.c2);
        if (n > 0) {                                     // the previous output product has read its exponentials
          ok = __all_sync(0xffffffffu, mbar_wait(p_free, (n - 1u) & 1u, 47));
          if (!ok) break;
          tc_fence_after();
        }
        if (kb == 0) {
          m = mx;
        } else {
          const bool raise = mx - m > kLazy;             // -inf so far: true as soon as a finite score comes
          if (__any_sync(0xffffffffu, raise)) {
            const float f = raise ? attn::ex2_approx(m - mx) : 1.f;
            if (raise) m = mx;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < P / 32; ++c) {
              uint32_t r[32];
              tmem_ld32_nowait(to + c * 32, r);
              attn::tmem_ld_wait32(r);
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
              attn::tmem_st32(to + c * 32, r);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        if (near) l += mask ? row_exp<true, true>(ts, tp, bp, 0.f, ref, lim, p.c.c2) : row_exp<true, false>(ts, tp, bp, 0.f, ref, lim, p.c.c2);
        else l += mask ? row_exp<false, true>(ts, tp, bp, flat, ref, lim, p.c.c2) : row_exp<false, false>(ts, tp, bp, flat, ref, lim, p.c.c2);
        attn::tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (!ok) break;
      sb_half* out = reinterpret_cast<sb_half*>(p.out.p) + (long long)w.h * p.out.sH + (long long)w.b * p.out.sB + (long long)j * p.out.sR;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (w.tiles > 0) {
        if (lane == 0) mbar_arrive(b_empty + 8 * bb);
        ok = __all_sync(0xffffffffu, mbar_wait(p_free, (n - 1u) & 1u, 47));
        if (!ok) break;
        tc_fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < P / 32; ++c) {
        uint32_t r[32];
        if (w.tiles > 0) {
          tmem_ld32_nowait(to + c * 32, r);
          attn::tmem_ld_wait32(r);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (row && c * 32 < p.c.P) store_features(out + c * 32 * p.out.sP, p.out.sP, r, inv, min(32, p.c.P - c * 32));
      }
      if (row && p.lse.p)
        p.lse.p[(long long)w.h * p.lse.sH + (long long)w.b * p.lse.sB + (long long)j * p.lse.sJ] =
            l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
      if (w.tiles > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
        ++it;
      }
    }
  }
  flash::drain_after_error();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
  }
}

}  // namespace rel
