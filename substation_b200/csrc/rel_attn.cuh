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

constexpr int kPad = 96;                             // 64 columns and the 32 rows of a warp
constexpr float kLazy = 8.f;                         // log2 units a row's reference may lag behind its maximum
// The forward pass' exponentials are times 2^kRaise, as far up as float16 goes beside that, so that many small ones do not vanish in it:
// steps are 2^-31 of the reference's exponential instead of 2^-24.
constexpr float kRaise = kRelScaled ? 15.f - kLazy : 0.f;

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
// D (+)= A * B, A in shared memory or (ts) in tensor memory as 16-bit pairs, a row per lane.  The whole warp comes here and one
// thread issues (`on`), so that the operands are the warp's and not a branch's.
__device__ __forceinline__ void umma_ss(uint32_t on, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 e, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t on, uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 e, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar), "r"(on) : "memory");
}
// A value that all lanes hold, as the compiler can see.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {   // (no wait)
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ float2 pair(const uint32_t* r, int i) { return make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])); }
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
__device__ __forceinline__ void mma_rows(uint32_t on, uint32_t d, uint32_t a, uint32_t b) {
  const uint32_t idesc = (1u << 4) | SB_IDESC_AB_FMT | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
  const uint64_t da = make_desc(a, 16u, 1024u), db = make_desc(b, 16u, 1024u);
#pragma unroll
  for (int k = 0; k < P / 16; ++k)
    umma_ss(on, d, da + (uint64_t)((k >> 2) * (128 * 8) + (k & 3) * 2), db + (uint64_t)((k >> 2) * (N * 8) + (k & 3) * 2), idesc,
             k > 0 ? 1u : 0u);
}
// D[128 x P] (+)= S[128 x K] * B, S in tensor memory and B [K rows x P features] in shared memory
template <int P, int K>
__device__ __forceinline__ void mma_weighted(uint32_t on, uint32_t d, uint32_t s, uint32_t b, bool accumulate) {
  const uint32_t idesc = (1u << 4) | SB_IDESC_AB_FMT | (1u << 16) | ((uint32_t)(P >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
  const uint64_t db = make_desc(b, (uint32_t)(K * 128), 1024u);
#pragma unroll
  for (int k = 0; k < K / 16; ++k)
    umma_ts(on, d, s + (uint32_t)(k * 8), db + (uint64_t)(k * 128), idesc, (accumulate || k > 0) ? 1u : 0u);
}
// D[128 x P] = S^T * B, S [128 x 128] in shared memory as two boxes of 64 columns, summed over its rows, B [128 rows x P features]
template <int P>
__device__ __forceinline__ void mma_transposed(uint32_t on, uint32_t d, uint32_t s, uint32_t b) {
  const uint32_t idesc = (1u << 4) | SB_IDESC_AB_FMT | (1u << 15) | (1u << 16) | ((uint32_t)(P >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
  const uint64_t da = make_desc(s, 16384u, 1024u), db = make_desc(b, 16384u, 1024u);
#pragma unroll
  for (int k = 0; k < 8; ++k) umma_ss(on, d, da + (uint64_t)(k * 128), db + (uint64_t)(k * 128), idesc, k > 0 ? 1u : 0u);
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
// 32 accumulator columns -> alpha * value, 16-bit, the first n of them, at ptr[p * sP].  A thread writes its own row, whole sectors
// at a time where the row allows it.
__device__ __forceinline__ void store_features(sb_half* ptr, long long sP, const uint32_t* r, float alpha, int n) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(ptr);
  if (sP == 1 && (at & 15u) == 0 && (n & 7) == 0) {
    uint32_t o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = flash::pack2(__uint_as_float(r[2 * e]) * alpha, __uint_as_float(r[2 * e + 1]) * alpha);
    if ((at & 31u) == 0 && n == 32) {
#pragma unroll
      for (int v = 0; v < 2; ++v)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr + v * 16), "r"(o[8 * v]), "r"(o[8 * v + 1]), "r"(o[8 * v + 2]),
                     "r"(o[8 * v + 3]), "r"(o[8 * v + 4]), "r"(o[8 * v + 5]), "r"(o[8 * v + 6]), "r"(o[8 * v + 7]) : "memory");
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (v * 8 < n) reinterpret_cast<uint4*>(ptr)[v] = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < n) ptr[e * sP] = sb_f2h(__uint_as_float(r[e]) * alpha);
  }
}

// 32 accumulator columns of a warp's 32 rows -> alpha * value, 16-bit: the first `features` of the first `rows` rows, at
// ptr[row * sR + feature * sP], by way of 2 KB of shared memory.  Four lanes write 64 bytes of a row; a thread writing its own row
// meets 32 lines with each instruction, which counts where items are short (training at B=96, L=128: 121 us with threads' own rows, 116
// so); elsewhere the registers that this takes cost more (forward at B=16, L=384: 28.6 -> 29.9 us).
constexpr int kStoreBytes = 2048;
__device__ __forceinline__ void store_rows(uint8_t* mem, sb_half* ptr, long long sR, long long sP, const uint32_t* r, float alpha, int features,
                                           int rows, int lane) {
#pragma unroll
  for (int v = 0; v < 4; ++v) {                          // 16-byte piece v of row `lane` at v ^ (lane / 2 & 3)
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = flash::pack2(__uint_as_float(r[v * 8 + 2 * e]) * alpha, __uint_as_float(r[v * 8 + 2 * e + 1]) * alpha);
    *reinterpret_cast<uint4*>(mem + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)) = o;
  }
  __syncwarp();
  if (sP == 1 && ((reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(2 * sR)) & 15u) == 0 && (features & 7) == 0) {
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + (lane >> 2);
      if (row < rows && piece * 8 < features)
        *reinterpret_cast<uint4*>(ptr + row * sR + piece * 8) = *reinterpret_cast<const uint4*>(mem + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
    }
  } else if (lane < rows) {
    const sb_half* row = reinterpret_cast<const sb_half*>(mem + lane * 64);
    sb_half* out = ptr + lane * sR;
#pragma unroll 1
    for (int f = 0; f < features; ++f, out += sP) *out = row[(((f >> 3) ^ ((lane >> 1) & 3)) << 3) + (f & 7)];
  }
  __syncwarp();
}

// ---- work items ------------------------------------------------------------------------------------------------
// Items come from a counter in memory, so that long ones do not hold up others (which item runs where changes nothing in its
// results).  The producer warp works out an item's sizes, once, and hands them to the other warps through kSlots places in shared
// memory: 48 bytes each, {kind, b, h, t}, {first, keys, tiles, each}, {t0}; kind < 0 ends.
constexpr int kSlots = 4;
struct Item {
  int kind, b, h, t;
  int first, keys, tiles, each;
  int t0;
};
__device__ __forceinline__ void write_item(uint8_t* slot, const Item& w) {
  reinterpret_cast<int4*>(slot)[0] = make_int4(w.kind, w.b, w.h, w.t);
  reinterpret_cast<int4*>(slot)[1] = make_int4(w.first, w.keys, w.tiles, w.each);
  reinterpret_cast<int*>(slot)[8] = w.t0;
}
__device__ __forceinline__ void read_item(const uint8_t* slot, Item* w) {
  const int4 a = reinterpret_cast<const int4*>(slot)[0], b = reinterpret_cast<const int4*>(slot)[1];
  w->kind = a.x; w->b = a.y; w->h = a.z; w->t = a.w;
  w->first = b.x; w->keys = b.y; w->tiles = b.z; w->each = b.w;
  w->t0 = reinterpret_cast<const int*>(slot)[8];
}
// The next item for a consuming warp; false at the end, or with *ok = false when a wait ran out.
__device__ __forceinline__ bool take_item(const uint8_t* slots, uint32_t full, uint32_t empty, uint32_t* taken, int lane, Item* w, bool* ok) {
  const uint32_t s = *taken & (kSlots - 1u);
  *ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * s, (*taken / kSlots) & 1u, 51));
  if (!*ok) return false;
  read_item(slots + 48 * s, w);
  __syncwarp();
  if (lane == 0) mbar_arrive(empty + 8 * s);
  ++*taken;
  return w->kind >= 0;
}
// The producer's side: publishes item `w` (or the end).
__device__ __forceinline__ bool put_item(uint8_t* slots, uint32_t full, uint32_t empty, uint32_t* put, int lane, const Item& w) {
  const uint32_t s = *put & (kSlots - 1u);
  if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((*put / kSlots) & 1u) ^ 1u, 52))) return false;
  if (lane == 0) {
    write_item(slots + 48 * s, w);
    mbar_arrive(full + 8 * s);
  }
  __syncwarp();
  ++*put;
  return true;
}

// ---- forward ---------------------------------------------------------------------------------------------------
constexpr int kFwdThreads = 224;                     // producer warp, two MMA warps, four softmax warps

struct FwdParams {
  Common c;
  int nq, units, chunk;                              // query tiles of a unit; units = H * B; units taken together
  int items;
  int* next;                                         // work queue
  Proj out;
  RelRows lse;
};

// The i-th work item: a tile of queries of one head and sample.  Units go in chunks, and within a chunk the last tiles first:
// with a causal span these are the long ones, and one head's keys stay in L2 while its tiles are worked on.
__device__ __forceinline__ Item fwd_item(const FwdParams& p, int i) {
  Item it;
  it.kind = 0; it.each = it.t0 = 0;
  const int per = p.chunk * p.nq, c = i / per, r = i % per;
  const int here = min(p.chunk, p.units - c * p.chunk), unit = c * p.chunk + r % here;
  it.t = p.nq - 1 - r / here;
  it.b = unit / p.c.H;
  it.h = unit % p.c.H;
  it.first = first_of(p.c, it.b);
  it.keys = keys_of(p.c, it.b);
  if (p.c.causal) it.keys = max(0, min(it.keys, it.first + min(p.c.J, it.t * 128 + 128)));
  it.tiles = (it.keys + 63) >> 6;
  return it;
}

// Tiles of 64 keys.  Tensor memory: two buffers of scores (64 columns each), which their exponentials overwrite, then the output.
// Shared memory of a CTA (two per SM): query tiles, the ring of key and value tiles, two rows of biases, barriers.
template <int P>
struct FwdCfg {
  static constexpr int kN = 64;
  static constexpr uint32_t kO = 2 * kN;
  static constexpr int kQTile = 128 * P * 2, kTile = kN * P * 2;
  static constexpr int kQ = P == 64 ? 2 : 1;         // query tiles (the next item's is fetched early)
  static constexpr int kRing = P == 64 ? 8 : 4;
  static constexpr int kTiles = kQ * kQTile + kRing * kTile;
  static constexpr int smem(int pitch) { return kTiles + 2 * pitch * 4 + 1024 + 128 + 16 * kRing + 16 * kSlots + 48 * kSlots + 16; }
};

// A row's state: reference of its exponentials, their sum so far.
struct Row { float m, l; };

// The reference rises: what stands in tensor memory, the output (where `started`) and the tile's first `chunks` chunks of
// exponentials, is brought to it.  Rare.
template <int P>
__device__ __noinline__ void rescale(uint32_t to, uint32_t tp, bool started, int chunks, float f) {
  if (started) {
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
  attn::tmem_st_wait();
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    uint32_t r[16];
    tmem_ld16(tp + c * 16, r);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float2 v = sb_h22f2(*reinterpret_cast<const sb_half2*>(&r[e]));
      r[e] = flash::pack2(v.x * f, v.y * f);
    }
    tmem_st16(tp + c * 16, r);
  }
  attn::tmem_st_wait();
}

// A thread's row of 64 scores, 32 columns at a time while the next 32 are on their way: exponentials against the row's
// reference as 16-bit pairs, which overwrite scores already read.  `settled` waits for the output.  The reference lags behind the
// maximum by at most 2^kLazy; a chunk that exceeds it makes it rise before its own exponentials are taken.  Exponentials of the tile's
// first chunk, if there are any, are then rounded a second time.  (References that rise by whole powers of two would avoid that, but then
// the row's largest exponential is rounded too, which is 1 otherwise: rows that one key rules lose more.)
// NEAR: the bias varies, bp[c] is column c's; else it is `flat`.  MASK: columns from lim on are hidden.
template <int P, bool NEAR, bool MASK, class Settled>
__device__ __forceinline__ void row_tile(uint32_t s, uint32_t to, bool started, const float* bp, float flat, int lim, float c2, Row& row,
                                         Settled&& settled) {
  float2 sum = make_float2(0.f, 0.f);
  const float2 c22 = make_float2(c2, c2);
  auto chunk = [&](int c, uint32_t* r, uint32_t* coming) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float2 t = pair(r, e);
      if (NEAR) t = fma2(t, c22, make_float2(bp[c * 32 + e], bp[c * 32 + e + 1]));
      if (MASK) {
        if (c * 32 + e >= lim) t.x = -INFINITY;
        if (c * 32 + e + 1 >= lim) t.y = -INFINITY;
      }
      if (NEAR || MASK) {
        r[e] = __float_as_uint(t.x);
        r[e + 1] = __float_as_uint(t.y);
      }
      mx[(e >> 1) & 3] = fmaxf(fmaxf(mx[(e >> 1) & 3], t.x), t.y);
    }
    float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    if (!NEAR && m > -INFINITY) m = fmaf(m, c2, flat);
    if (!started && c == 0) {
      row.m = m;
    } else {
      const bool raise = m - row.m > kLazy;              // no finite score so far: true as soon as one comes
      if (__any_sync(0xffffffffu, raise)) {
        const float f = raise ? attn::ex2_approx(row.m - m) : 1.f;
        if (raise) row.m = m;
        row.l *= f;
        sum.x *= f;
        sum.y *= f;
        attn::tmem_ld_wait32(coming);                    // (a call moves registers)
        settled();
        rescale<P>(to, s, started, c, f);
      }
    }
    const float ref = row.m == -INFINITY ? 0.f : row.m;
    const float2 off = make_float2((NEAR ? kRaise : flat + kRaise) - ref, (NEAR ? kRaise : flat + kRaise) - ref);
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float2 x = NEAR ? add2(pair(r, e), off) : fma2(pair(r, e), c22, off);
      x.x = attn::ex2_approx(x.x);
      x.y = attn::ex2_approx(x.y);
      sum = add2(sum, x);
      w[e >> 1] = flash::pack2(x.x, x.y);
    }
    tmem_st16(s + c * 16, w);
  };
  uint32_t ra[32], rb[32];
  tmem_ld32_nowait(s, ra);
  attn::tmem_ld_wait32(ra);
  tmem_ld32_nowait(s + 32, rb);
  chunk(0, ra, rb);
  attn::tmem_ld_wait32(rb);
  chunk(1, rb, ra);
  row.l += sum.x + sum.y;
}

// One CTA: 128 queries of one unit against its keys, one pass with running references and sums; two CTAs per SM.  Scores are
// multiplied a tile ahead of the softmax, by a warp of their own: with one warp for both products and one buffer, issuing and
// handing over took most of the time.  Exponentials go back into tensor memory as 16-bit pairs (rounded once, as an operand of the
// second product has to be), where that product takes them from.  Softmax warps: thread = row.
// Calls, with the rows of biases, replayed from a graph: B=2, L=4096, 16 heads of 64 (137 GFLOP) 242 us, 35 % of the measured matrix rate;
// B=8, L=512: 26 us; B=2, L=2000 causal, 16 heads of 128 on 4: 53 us.  Bound by the softmax warps, of which a scheduler has two:
// exponentials keep their unit busy for 53 % of the time (without any 20 % less), half of it per tile of 64 columns is waiting for one's
// own results; without softmax 140 us.
template <int P>
__global__ void __launch_bounds__(kFwdThreads, 2)
rel_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
               const __grid_constant__ FwdParams p) {
  using Cfg = FwdCfg<P>;
  constexpr int kRing = Cfg::kRing, kQ = Cfg::kQ, N = Cfg::kN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sq = (raw + 1023u) & ~1023u, ring = sq + kQ * Cfg::kQTile;
  const uint32_t sbias = sq + Cfg::kTiles, bars = sbias + 2u * p.c.pitch * 4u;
  const uint32_t q_full = bars, q_empty = bars + 16, s_full = bars + 32, p_full = bars + 48, o_empty = bars + 64;
  const uint32_t b_full = bars + 80, b_empty = bars + 96, p_free = bars + 112, kv_full = bars + 128, kv_empty = kv_full + 8 * kRing, item_full = kv_empty + 8 * kRing, item_empty = item_full + 8 * kSlots;
  uint8_t* gen = smem_raw + (sq - raw);
  const float* bias_s = reinterpret_cast<const float*>(gen + (sbias - sq));
  uint8_t* slots = gen + (item_empty + 8 * kSlots - sq);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(slots + 48 * kSlots);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_empty + 8 * i, 4);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(p_free + 8 * i, 1);
    }
    mbar_init(o_empty, 4);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(item_full + 8 * i, 1);
      mbar_init(item_empty + 8 * i, 6);
    }
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
  const uint32_t tmem = uniform(*reinterpret_cast<volatile uint32_t*>(tmem_slot));
  grid_dependency_sync();

  // `it` counts the items that see a key, n their key tiles
  uint32_t taken = 0;
  auto take = [&](Item* w, bool* ok) { return take_item(slots, item_full, item_empty, &taken, lane, w, ok); };
  if (warp == 0) {
    // ---------------- producer: queries and biases of the item, then its keys and values in turn ----------------
    uint32_t it = 0, x = 0, put = 0;
    bool ok = true;
    int id = blockIdx.x;
    while (ok) {
      int after = 0;
      if (lane == 0 && id < p.items) after = atomicAdd(p.next, 1) + (int)gridDim.x;
      Item w;
      w.kind = -1;
      if (id < p.items) w = fwd_item(p, id);
      ok = put_item(slots, item_full, item_empty, &put, lane, w);
      if (!ok || id >= p.items) break;
      id = __shfl_sync(0xffffffffu, after, 0);
      if (w.tiles == 0) continue;
      const uint32_t qb = it % kQ, bb = it & 1u;
      ok = __all_sync(0xffffffffu, mbar_wait(q_empty + 8 * qb, ((it / kQ) & 1u) ^ 1u, 41)) &&
           __all_sync(0xffffffffu, mbar_wait(b_empty + 8 * bb, ((it >> 1) & 1u) ^ 1u, 41));
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(q_full + 8 * qb, Cfg::kQTile);
        load_rows<P, 128>(sq + qb * Cfg::kQTile, &tmQ, q_full + 8 * qb, w.t * 128, w.h, w.b);
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
          load_rows<P, N>(ring + s * Cfg::kTile, i & 1 ? &tmV : &tmK, kv_full + 8 * s, (i >> 1) * N, hk, w.b);
        }
        __syncwarp();
      }
      ++it;
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer of scores, a tile ahead of the softmax ----------------
    const uint32_t on = flash::elect_one() ? 1u : 0u;
    uint32_t it = 0, n = 0;                              // ring uses are 2 n (keys) and 2 n + 1 (values)
    bool ok = true;
    Item w;
    while (ok && take(&w, &ok)) {
      if (w.tiles == 0) continue;
      const uint32_t qb = it % kQ;
      ok = __all_sync(0xffffffffu, mbar_wait(q_full + 8 * qb, (it / kQ) & 1u, 42));
      const int tiles = uniform(w.tiles);
      for (int i = 0; i < tiles && ok; ++i, ++n) {
        const uint32_t s = 2 * n % kRing, sb = n & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(kv_full + 8 * s, (2 * n / kRing) & 1u, 42) && mbar_wait(p_free + 8 * sb, ((n >> 1) & 1u) ^ 1u, 42));
        if (!ok) break;
        tc_fence_after();
        mma_rows<P, N>(on, tmem + sb * N, sq + qb * Cfg::kQTile, ring + s * Cfg::kTile);
        commit_if(on, s_full + 8 * sb);
        commit_if(on, kv_empty + 8 * s);
        if (i == tiles - 1) commit_if(on, q_empty + 8 * qb);
      }
      ++it;
    }
  } else if (warp == 2) {
    // ---------------- MMA issuer of the output ----------------
    const uint32_t on = flash::elect_one() ? 1u : 0u;
    uint32_t it = 0, n = 0;
    bool ok = true;
    Item w;
    while (ok && take(&w, &ok)) {
      if (w.tiles == 0) continue;
      const int tiles = uniform(w.tiles);
      for (int i = 0; i < tiles; ++i, ++n) {
        const uint32_t s = (2 * n + 1) % kRing, sb = n & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(kv_full + 8 * s, ((2 * n + 1) / kRing) & 1u, 43));
        if (ok && w.keys - i * N < N) zero_rows<P, N>(gen + (ring - sq) + s * Cfg::kTile, w.keys - i * N, lane);
        ok = ok && __all_sync(0xffffffffu, mbar_wait(p_full + 8 * sb, (n >> 1) & 1u, 43) && (i > 0 || mbar_wait(o_empty, (it & 1u) ^ 1u, 44)));
        if (!ok) break;
        tc_fence_after();
        mma_weighted<P, N>(on, tmem + Cfg::kO, tmem + sb * N, ring + s * Cfg::kTile, i > 0);
        commit_if(on, kv_empty + 8 * s);
        commit_if(on, p_free + 8 * sb);
      }
      ++it;
    }
  } else {
    // ---------------- softmax warps: thread = one query ----------------
    const int q = warp & 3;
    const int rt = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t to = tmem + lanes + Cfg::kO;
    uint32_t n = 0, it = 0;
    bool ok = true;
    Item w;
    while (ok && take(&w, &ok)) {
      const int j = w.t * 128 + rt, pos = w.first + j;
      const bool row = j < p.c.J;
      int mine = w.keys;                                 // keys that this row sees
      if (p.c.causal) mine = min(mine, pos + 1);
      Row state = {-INFINITY, 0.f};
      const uint32_t bb = it & 1u;
      const float* bias = bias_s + bb * p.c.pitch;
      if (w.tiles > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_full + 8 * bb, (it >> 1) & 1u, 45));
        if (!ok) break;
      }
      // columns of the tile that this row sees, the fewest of the warp's rows, the relative position of the first column at this
      // row, and the lowest of the warp's block (its highest is lo + N + 30)
      int lim = mine, least = __reduce_min_sync(0xffffffffu, mine), rel0 = -pos, lo = -(w.first + w.t * 128 + q * 32 + 31);
      for (int kb = 0; kb < w.tiles; ++kb, ++n, lim -= N, least -= N, rel0 += N, lo += N) {
        const uint32_t sb = n & 1u, ts = tmem + lanes + sb * N;
        const bool near = lo + N + 30 > -p.c.reach && lo < p.c.reach, mask = least < N;
        // outside the varying part, a place in the row where N entries have the end's value
        const float* bp = bias + (near ? rel0 + p.c.reach + kPad : lo >= p.c.reach ? kPad + 2 * p.c.reach : 0);
        const float flat = bp[0];
        ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * sb, (n >> 1) & 1u, 46));
        if (!ok) break;
        tc_fence_after();
        auto settled = [&] {                             // every product so far is in the output
          ok = kb == 0 || __all_sync(0xffffffffu, mbar_wait(p_free + 8 * ((n - 1u) & 1u), ((n - 1u) >> 1) & 1u, 47));
          tc_fence_after();
        };
        if (mask) row_tile<P, true, true>(ts, to, kb > 0, bp, 0.f, lim, p.c.c2, state, settled);
        else if (near) row_tile<P, true, false>(ts, to, kb > 0, bp, 0.f, lim, p.c.c2, state, settled);
        else row_tile<P, false, false>(ts, to, kb > 0, bp, flat, lim, p.c.c2, state, settled);
        if (!ok) break;
        attn::tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * sb);
      }
      if (!ok) break;
      sb_half* out = reinterpret_cast<sb_half*>(p.out.p) + (long long)w.h * p.out.sH + (long long)w.b * p.out.sB + (long long)j * p.out.sR;
      const float inv = sees_none(state.l) ? 0.f : 1.f / state.l;
      if (w.tiles > 0) {
        if (lane == 0) mbar_arrive(b_empty + 8 * bb);
        ok = __all_sync(0xffffffffu, mbar_wait(p_free + 8 * ((n - 1u) & 1u), ((n - 1u) >> 1) & 1u, 47));
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
            sees_none(state.l) ? -INFINITY : (state.m + (log2f(state.l) - kRaise)) * 0.6931471805599453f;
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

// ---- backward --------------------------------------------------------------------------------------------------
// producer warp, two MMA warps, two groups of four element warps, and in float16 a warp that puts the items' shifts into their biases
constexpr int kBwdThreads = kRelScaled ? 384 : 352;
constexpr int kRecord = 192;                         // floats of 64 query rows: log2-sum-exps, D, weights of the table's sums

struct BwdParams {
  Common c;
  int nq, nk;                                        // tiles of 128 queries, of 128 keys
  int first_q, items;                                // items below first_q: dK and dV of a key tile; the others: dQ of a query tile
  int chunk_k, chunk_q;
  int stages, held;                                  // ring of streamed pairs; held pairs (1 or 2)
  int sets;                                          // rows of sums per warp (1 or 2)
  float scale;
  const float* records;                              // [B][H][ceil(J / 64)][kRecord]
  const float* sizes;                                // float16: [B][H][ceil(J / 64)][8], but for BOTH the same again and [B][G][ceil(K / 64)][8]
  float* partial;                                    // [H][B * nq * 2][2 * reach + 1]
  int* next;                                         // work queue
  Proj dq, dk, dv;
};

// An item holds one pair of 128-row tiles and streams pairs of 64-row tiles past it: (K, V) held and (Q, dOUT) of every query
// head that shares them streamed (kind 0), or (Q, dOUT) held and (K, V) streamed (kind 1).  `b`, `h`, `t`: the held tile;
// `tiles` streamed ones, `each` from t0 on for each head in turn.
template <bool BOTH>
__device__ __forceinline__ Item bwd_item(const BwdParams& p, int i) {
  Item it;
  it.kind = !BOTH && i >= p.first_q ? 1 : 0;
  if (it.kind) i -= p.first_q;
  const int rows = it.kind ? p.nq : p.nk, heads = it.kind ? p.c.H : p.c.G, chunk = it.kind ? p.chunk_q : p.chunk_k;
  const int per = chunk * rows, c = i / per, r = i % per;
  const int here = min(chunk, heads * p.c.B - c * chunk), unit = c * chunk + r % here;
  it.t = it.kind ? rows - 1 - r / here : r / here;   // long ones first where the span is causal
  it.b = unit / heads;
  it.h = unit % heads;
  it.first = first_of(p.c, it.b);
  it.keys = keys_of(p.c, it.b);
  it.t0 = 0;
  if (it.kind) {
    if (p.c.causal) it.keys = max(0, min(it.keys, it.first + min(p.c.J, it.t * 128 + 128)));
    it.each = it.tiles = (it.keys + 63) >> 6;
  } else {
    const int all = (p.c.J + 63) >> 6;
    if (p.c.causal && !BOTH) it.t0 = min(all, max(0, it.t * 128 - it.first) >> 6);
    it.each = it.t * 128 < it.keys ? all - it.t0 : 0;
    it.tiles = it.each * (p.c.H / p.c.G);
  }
  return it;
}

// float16: an item's score gradients are rounded to 16 bits times 2^shift, its softmax weights times 2^max(shift, 0), which results lose
// again.  A weight w is at most one, so that a shift of at most 15 keeps it.  A score gradient is w (dP - D) = w dout (v - out), at most
// N = |dout| (|v| + |out|) with the longest rows that the item meets (dK and dV sum over them, so they share a factor): times 2^15 over
// the next power of two from N on it is held.  An item of queries has the v of all its keys, which bound its out; then the difference is one
// of two values of dP, at most |dout| |v| each, times w (1 - w), which is half that at most.  So what is looked at for an item grows as
// its own work does.  (A tight bound counts: largest magnitudes instead of norms gave shifts smaller by 4 to 5, with which keys of
// a weight below 1e-6 beside output gradients of 30 lost digits that their own dk could hold, for 2 us less.)

// The largest numbers of three lists, n[.] blocks of eight each, as the lane finds them; all three are on their way together.
__device__ __forceinline__ void largest_of(const float* const (&at)[3], const int (&n)[3], int lane, float (&m)[3]) {
  m[0] = m[1] = m[2] = 0.f;
#pragma unroll 1
  for (int i = lane; i < 2 * max(n[0], max(n[1], n[2])); i += 64) {
    float4 v[3][2];
#pragma unroll
    for (int x = 0; x < 3; ++x)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        v[x][k] = i + 32 * k < 2 * n[x] ? reinterpret_cast<const float4*>(at[x])[i + 32 * k] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < 3; ++x)
#pragma unroll
      for (int k = 0; k < 2; ++k) m[x] = fmaxf(m[x], fmaxf(fmaxf(v[x][k].x, v[x][k].y), fmaxf(v[x][k].z, v[x][k].w)));
  }
}
__device__ __forceinline__ float largest_in_warp(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }
// 2^top over the next power of two from the root of n2 on, 2^15 at most.  (n2: of float16's numbers 0, or from 2^-96 to 2^81)
__device__ __forceinline__ int item_shift(float n2, int top) { return n2 > 0.f ? min(15, top - (((int)(__float_as_uint(n2) >> 23) - 125) >> 1)) : 15; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// BOTH: units of one tile of queries and one of keys, each key head with one query head: an item gives all three gradients and
// everything is computed once.  dQ needs score gradients with the keys as the summed index, so they go to shared memory as
// well ([128 keys x 128 queries], 32 KB).
template <int P, bool BOTH>
struct BwdCfg {
  static_assert(P == 64 || !BOTH, "tensor memory has no room for a third accumulator of 128 columns");
  static constexpr int kHeld = 2 * 128 * P * 2 + 2048, kStream = 2 * 64 * P * 2, kStage = kStream + 1024;   // tiles and records
  static constexpr int kStaged = BOTH ? 32768 : 0;
  // Tensor memory: buffers of scores and dP (64 columns each), then the accumulators.  A third buffer, where it fits, lets a tile
  // be multiplied before either group is done with its own: without it a group waits for two products and two hand-overs.
  static constexpr int kBuf = P == 64 && !BOTH ? 3 : 2;
  static constexpr uint32_t kAcc = P == 64 ? 384 : 256, kAccQ = 256;
  static constexpr int smem(int stages, int held, int sets, int pitch, int reach) {
    return held * kHeld + stages * kStage + kStaged + (BOTH ? 8 * kStoreBytes : 0) + 2 * pitch * 4 + sets * 8 * ((2 * reach + 4) & ~3) * 4 + 1024 + 400 + 48 * kSlots + 32;
  }
};

// Scores and dP of a thread's row of 64 columns -> exponentials and score gradients, 16-bit pairs over the columns they came
// from, 32 columns at a time.  Column c has the bias bp[c] (key tiles: bp[-c]; NEAR) or `flat`.
// What differs between the two kinds of items: in key tiles (KEYS) a thread is a key, log-sum-exps and D change along columns
// (L, D in shared memory), visible columns are c >= lim; in query tiles a thread is a query and visible columns are c < lim.
// `emit` gets every score gradient, `block` is told after each 32 columns; `staged`: where the row goes in shared memory too.
// In masked tiles of keys score gradients are times `gf`, which their weights are not.
template <bool KEYS, bool NEAR, bool MASK, class Emit, class Block>
__device__ __forceinline__ void turn_tile(uint32_t ts, const float* bp, float flat, const float* L, const float* D, float lse, float dsum,
                                          int lim, float c2, Emit&& emit, Block&& block, uint8_t* staged = nullptr, int row7 = 0, float gf = 1.f) {
  const float2 c22 = make_float2(c2, c2), minus = make_float2(-1.f, -1.f);
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    uint32_t s[32], g[32], dm[16], pm[16];
    tmem_ld32_nowait(ts + c * 32, s);
    tmem_ld32_nowait(ts + 64 + c * 32, g);
    const float* bc = bp + (KEYS ? -c * 32 : c * 32);
    attn::tmem_ld_wait32(s);
    attn::tmem_ld_wait32(g);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      float4 l4 = make_float4(lse, lse, lse, lse), d4 = make_float4(dsum, dsum, dsum, dsum);
      if (KEYS) {
        l4 = *reinterpret_cast<const float4*>(L + c * 32 + e);
        d4 = *reinterpret_cast<const float4*>(D + c * 32 + e);
      }
#pragma unroll
      for (int x = 0; x < 4; x += 2) {
        const int i = e + x, col = c * 32 + i;
        const float2 l = x ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y), d = x ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);
        const float2 b = NEAR ? (KEYS ? make_float2(bc[-i], bc[-i - 1]) : make_float2(bc[i], bc[i + 1])) : make_float2(flat, flat);
        float2 pr = fma2(pair(s, i), c22, fma2(l, minus, b));
        pr.x = attn::ex2_approx(pr.x);
        pr.y = attn::ex2_approx(pr.y);
        float2 ds = mul2(pr, fma2(d, minus, pair(g, i)));
        if (kRelScaled && KEYS && MASK) ds = mul2(ds, make_float2(gf, gf));
        if (MASK) {
          const bool seen0 = KEYS ? col >= lim : col < lim, seen1 = KEYS ? col + 1 >= lim : col + 1 < lim;
          pr = make_float2(seen0 ? pr.x : 0.f, seen1 ? pr.y : 0.f);
          ds = make_float2(seen0 ? ds.x : 0.f, seen1 ? ds.y : 0.f);
        }
        emit(i, ds.x);
        emit(i + 1, ds.y);
        if (KEYS) pm[i >> 1] = flash::pack2(pr.x, pr.y);
        dm[i >> 1] = flash::pack2(ds.x, ds.y);
      }
    }
    if (KEYS) tmem_st16(ts + c * 16, pm);
    tmem_st16(ts + 64 + c * 16, dm);
    if (staged) {                                        // (a row of 128 bytes, 16-byte piece i at i ^ (row & 7))
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<uint4*>(staged + (((c * 4 + v) ^ row7) << 4)) = make_uint4(dm[4 * v], dm[4 * v + 1], dm[4 * v + 2], dm[4 * v + 3]);
    }
    block(c);
  }
}

// float16: the warp that finds the items' shifts.  Added to the biases of a key item they make its exponentials 2^shift times as large.
// A CTA's first item waits for that (and for every line of this code to be fetched, which is why it is short), later ones do not.  All
// that float16 has for its range, this warp and the sizes that row_records_kernel finds, takes 6.5 us of a forward and backward call at B=8,
// L=512 (109.2 -> 115.7), 5.5 at B=96, L=128 (116.1 -> 121.6), 4 at B=2, L=2000 causal with 128 features (270 -> 274), and nothing to be
// seen at B=2, L=4096.  One more multiplication for every score gradient of a key item, instead of shifted biases, took 2 us more
// at B=8 and 10 at L=4096; this warp's code behind the others' 1 to 4 us.
struct ShiftWarp {
  const uint8_t *slots, *held;
  float4* biases;                                    // two rows
  int* shifts;                                       // of the last four items with tiles
  uint32_t item_full, item_empty, h_full, b_full, b_ready;
};
template <int P, bool BOTH>
__device__ __forceinline__ void shift_warp(const BwdParams& p, const ShiftWarp& s) {
  const int lane = threadIdx.x & 31, rep = p.c.H / p.c.G, blocks = (p.c.J + 63) >> 6, blocks_v = (p.c.K + 63) >> 6;
  uint32_t taken = 0, live = 0, run = 0;
  bool ok = true;
  Item w;
  while (ok && take_item(s.slots, s.item_full, s.item_empty, &taken, lane, &w, &ok)) {
    if (w.tiles == 0) continue;
    const long long of_out = 8ll * p.c.B * p.c.H * blocks;
    const float* rows = p.sizes + 8 * (((long long)w.b * p.c.H + (w.kind ? w.h : w.h * rep)) * blocks + (w.kind ? 2 * w.t : 0));
    const float* values = p.sizes + 2 * of_out + 8 * (((long long)w.b * p.c.G + (w.kind ? w.h / rep : w.h)) * blocks_v + (w.kind ? 0 : 2 * w.t));
    const int n = w.kind ? min(2, blocks - 2 * w.t) : rep * blocks;
    float m[3];                                      // of dout, out, v: sums of squares
    largest_of({rows, rows + of_out, values}, {n, BOTH || w.kind ? 0 : n, BOTH ? 0 : w.kind ? (w.keys + 63) >> 6 : min(2, blocks_v - 2 * w.t)}, lane, m);
    if (BOTH) {                                      // the held values, 16 bytes at a time: their largest magnitude
      const uint32_t hb = p.held == 2 ? live & 1u : 0u, hp = p.held == 2 ? live >> 1 : live;
      ok = __all_sync(0xffffffffu, mbar_wait(s.h_full + 8 * hb, hp & 1u, 63));
      if (!ok) return;
      const uint4* tile = reinterpret_cast<const uint4*>(s.held + hb * BwdCfg<P, BOTH>::kHeld + 256 * P);
#pragma unroll 2
      for (int i = lane; i < w.keys * 8; i += 32) m[2] = fmaxf(m[2], finite_size(larger(half2_of(0u), tile[i])));
      m[2] *= m[2] * (float)p.c.P;
    }
    const float n2 = largest_in_warp(m[0]) * (largest_in_warp(m[1]) + largest_in_warp(m[2]));
    const int shift = BOTH || w.kind ? item_shift(n2, 16) : item_shift(2.f * n2, 15);   // ((|v| + |out|)^2 is at most 2 |v|^2 + 2 |out|^2)
    for (int done = 0; done < w.tiles; done += w.each, ++run) {
      ok = __all_sync(0xffffffffu, mbar_wait(s.b_full + 8 * (run & 1u), (run >> 1) & 1u, 63));
      if (!ok) return;
      // (four items before, whose place this is: its results were stored before the run but one before this began)
      if (lane == 0 && done == 0) s.shifts[live & 3u] = shift;
      if (!w.kind) {                                 // (query items have the log-sum-exps in registers)
        float4* row = s.biases + (run & 1u) * (p.c.pitch / 4);
        const float add = (float)max(shift, 0);
#pragma unroll 1
        for (int i = lane; i < p.c.pitch / 4; i += 32) {
          const float4 v = row[i];
          row[i] = make_float4(v.x + add, v.y + add, v.z + add, v.w + add);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(s.b_ready + 8 * (run & 1u));
    }
    ++live;
  }
}

// One CTA per SM.  The two groups of element warps take the streamed tiles in turn: while one turns scores and dP into
// exponentials and score gradients, the tensor cores multiply for the other.  Both results go back into tensor memory as 16-bit
// pairs, rounded once as operands have to be, where the second products take them from.  Everything is
// computed twice, once per kind of item (but for BOTH); the alternative, dQ summed over key tiles in memory, needs atomics whose order
// changes the result, or a partial dQ for every key tile.
// Calls, with records and the table's last sums, replayed from a graph: B=2, L=4096, 16 heads of 64 (344 GFLOP needed, 481 multiplied, as
// scores and dP are computed twice) 666 us, 32 % of the measured matrix rate on what is needed (forward and backward together 904 in that
// run); B=2, L=2000 causal, 16 heads of 128 on 4: 218 us; B=8, L=512: 83 us; BOTH at B=96, L=128: 88 us, bound by its items' beginnings
// and ends.  This kernel alone, where it took 658 us: without element work 410, without products 599: the element warps' instructions,
// two warps per scheduler.  A third group (128 registers a thread) took 694 us, scores from tensor memory 630 at best.
// The table's gradient: a score gradient belongs to its relative position, a diagonal of the tile.  A warp moves each column of
// its 32 x 32 blocks so that lane l holds diagonals l and l - 32 (one shuffle a column), adds the sums of a block to its own row
// of sums over relative positions, and a group of warps adds up its four rows per item.  Tiles outside the varying part of the
// bias have one sum.  Everything in a fixed order.
template <int P, bool BOTH>
__global__ void __launch_bounds__(kBwdThreads, 1)
rel_bwd_kernel(const __grid_constant__ CUtensorMap tmQh, const __grid_constant__ CUtensorMap tmGh, const __grid_constant__ CUtensorMap tmKh,
               const __grid_constant__ CUtensorMap tmVh, const __grid_constant__ CUtensorMap tmQs, const __grid_constant__ CUtensorMap tmGs,
               const __grid_constant__ CUtensorMap tmKs, const __grid_constant__ CUtensorMap tmVs, const __grid_constant__ BwdParams p) {
  using Cfg = BwdCfg<P, BOTH>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sheld = (raw + 1023u) & ~1023u, ring = sheld + p.held * Cfg::kHeld;
  const uint32_t staged = ring + p.stages * Cfg::kStage, sstore = staged + Cfg::kStaged, sbias = sstore + (BOTH ? 8 * kStoreBytes : 0);
  const int width = (2 * p.c.reach + 4) & ~3;        // floats of a warp's row of sums
  const uint32_t ssums = sbias + 2u * p.c.pitch * 4u, bars = ssums + p.sets * 8u * width * 4u;
  const uint32_t item_full = bars, item_empty = bars + 32, h_full = bars + 64, h_empty = bars + 80, b_full = bars + 96, b_empty = bars + 112;
  const uint32_t s_full = bars + 128, pd_full = bars + 152, acc_full = bars + 176, acc_empty = bars + 184, full = bars + 192, empty = bars + 256;
  uint8_t* gen = smem_raw + (sheld - raw);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + (bars + 320 - sheld));
  uint8_t* slots = gen + (bars + 400 - sheld);
  const uint32_t g_sync = bars + 352, buf_free = bars + 368, q_free = bars + 392, b_ready = kRelScaled ? bars + 400 + 48 * kSlots : b_full;
  int* shifts = reinterpret_cast<int*>(slots + 48 * kSlots + 16);   // of the last four items with tiles
  const float* bias_s = reinterpret_cast<const float*>(gen + (sbias - sheld));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(item_full + 8 * i, 1);
      mbar_init(item_empty + 8 * i, kBwdThreads / 32 - 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(h_full + 8 * i, 1);
      mbar_init(h_empty + 8 * i, 9);                   // the products, and the element warps, which read records
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_empty + 8 * i, 8);
      mbar_init(g_sync + 8 * i, 4);
      if (kRelScaled) mbar_init(b_ready + 8 * i, 1);
    }
    for (int i = 0; i < Cfg::kBuf; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(pd_full + 8 * i, 4);
      mbar_init(buf_free + 8 * i, 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 8);
    mbar_init(q_free, 1);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  {
    float* sums = reinterpret_cast<float*>(gen + (ssums - sheld));
    for (int i = threadIdx.x; i < p.sets * 8 * width; i += kBwdThreads) sums[i] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*reinterpret_cast<volatile uint32_t*>(tmem_slot));
  grid_dependency_sync();

  uint32_t taken = 0;
  auto take = [&](Item* w, bool* ok) { return take_item(slots, item_full, item_empty, &taken, lane, w, ok); };

  if (kRelScaled && warp == 11) {
    shift_warp<P, BOTH>(p, ShiftWarp{slots, gen, reinterpret_cast<float4*>(gen + (sbias - sheld)), shifts, item_full, item_empty, h_full, b_full, b_ready});
  } else if (warp == 0) {
    // ---------------- producer ----------------
    // live: items with tiles; run: tiles of one head in an item, which share a row of biases
    uint32_t put = 0, live = 0, run = 0, st = 0, st_phase = 1;
    const int rep = p.c.H / p.c.G, blocks = (p.c.J + 63) >> 6;
    bool ok = true;
    int id = blockIdx.x;
    while (ok) {
      int after = 0;
      if (lane == 0 && id < p.items) after = atomicAdd(p.next, 1) + (int)gridDim.x;
      Item w;
      w.kind = -1;
      if (id < p.items) w = bwd_item<BOTH>(p, id);
      ok = put_item(slots, item_full, item_empty, &put, lane, w);
      if (!ok || id >= p.items) break;
      if (w.tiles > 0) {
        const uint32_t hb = p.held == 2 ? live & 1u : 0u, hp = p.held == 2 ? live >> 1 : live;
        ok = __all_sync(0xffffffffu, mbar_wait(h_empty + 8 * hb, (hp & 1u) ^ 1u, 53));
        if (!ok) break;
        if (lane == 0) {
          const uint32_t d = sheld + hb * Cfg::kHeld;
          const int rows = min(2, blocks - w.t * 2) * kRecord * 4;   // bytes of a query tile's records
          mbar_expect_tx(h_full + 8 * hb, 512 * P + (w.kind ? rows : 0));
          load_rows<P, 128>(d, w.kind ? &tmQh : &tmKh, h_full + 8 * hb, w.t * 128, w.h, w.b);
          load_rows<P, 128>(d + 256 * P, w.kind ? &tmGh : &tmVh, h_full + 8 * hb, w.t * 128, w.h, w.b);
          if (w.kind) bulk_load(d + 512 * P, p.records + (((long long)w.b * p.c.H + w.h) * blocks + w.t * 2) * kRecord, rows, h_full + 8 * hb);
        }
        __syncwarp();
        ++live;
      }
      int head = w.kind ? w.h : w.h * rep, t = w.t0, left = w.each;
      for (int i = 0; i < w.tiles && ok; ++i) {
        if (left == w.each) {
          const uint32_t bb = run & 1u;
          ok = __all_sync(0xffffffffu, mbar_wait(b_empty + 8 * bb, ((run >> 1) & 1u) ^ 1u, 54));
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(b_full + 8 * bb, p.c.pitch * 4);
            bulk_load(sbias + bb * p.c.pitch * 4, p.c.bias_rows + (long long)head * p.c.pitch, p.c.pitch * 4, b_full + 8 * bb);
          }
          __syncwarp();
          ++run;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * st, st_phase, 55));
        if (!ok) break;
        if (lane == 0) {
          const uint32_t d = ring + st * Cfg::kStage, bar = full + 8 * st;
          mbar_expect_tx(bar, Cfg::kStream + (w.kind ? 0 : BOTH ? 768 : 512));
          if (w.kind) {
            load_rows<P, 64>(d, &tmKs, bar, t * 64, w.h / rep, w.b);
            load_rows<P, 64>(d + Cfg::kStream / 2, &tmVs, bar, t * 64, w.h / rep, w.b);
          } else {
            load_rows<P, 64>(d, &tmQs, bar, t * 64, head, w.b);
            load_rows<P, 64>(d + Cfg::kStream / 2, &tmGs, bar, t * 64, head, w.b);
            bulk_load(d + Cfg::kStream, p.records + (((long long)w.b * p.c.H + head) * blocks + t) * kRecord, BOTH ? 768 : 512, bar);
          }
        }
        __syncwarp();
        if (++st == (uint32_t)p.stages) { st = 0; st_phase ^= 1u; }
        ++t;
        if (--left == 0) { ++head; t = w.t0; left = w.each; }
      }
      id = __shfl_sync(0xffffffffu, after, 0);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer of scores and dP ----------------
    const uint32_t on = flash::elect_one() ? 1u : 0u;
    uint32_t live = 0, st = 0, st_phase = 0, bf = 0, bf_phase = 1;
    bool ok = true;
    Item w;
    while (ok && take(&w, &ok)) {
      if (w.tiles == 0) continue;
      const uint32_t hb = p.held == 2 ? live & 1u : 0u, hp = p.held == 2 ? live >> 1 : live, hd = sheld + hb * Cfg::kHeld;
      ok = __all_sync(0xffffffffu, mbar_wait(h_full + 8 * hb, hp & 1u, 56));
      const int tiles = uniform(w.tiles);
      for (int i = 0; i < tiles && ok; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * st, st_phase, 56) && mbar_wait(buf_free + 8 * bf, bf_phase, 56));
        if (!ok) break;
        tc_fence_after();
        const uint32_t x = ring + st * Cfg::kStage, ts = tmem + bf * 128u;
        if (w.kind && w.keys - i * 64 < 64) zero_rows<P, 64>(gen + (x - sheld), w.keys - i * 64, lane);
        if (BOTH && i == 0 && w.keys < 128) zero_rows<P, 128>(gen + (hd - sheld), w.keys, lane);
        mma_rows<P, 64>(on, ts, hd, x);
        mma_rows<P, 64>(on, ts + 64u, hd + 256 * P, x + Cfg::kStream / 2);
        commit_if(on, s_full + 8 * bf);
        if (++st == (uint32_t)p.stages) { st = 0; st_phase ^= 1u; }
        if (++bf == (uint32_t)Cfg::kBuf) { bf = 0; bf_phase ^= 1u; }
      }
      ++live;
    }
  } else if (warp == 2) {
    // ---------------- MMA issuer of the products that read what became of them ----------------
    const uint32_t on = flash::elect_one() ? 1u : 0u;
    uint32_t live = 0, st = 0, bf = 0, bf_phase = 0;
    bool ok = true;
    Item w;
    while (ok && take(&w, &ok)) {
      if (w.tiles == 0) continue;
      const int tiles = uniform(w.tiles), kind = uniform(w.kind);
      for (int i = 0; i < tiles; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait(pd_full + 8 * bf, bf_phase, 57) && (i > 0 || mbar_wait(acc_empty, (live & 1u) ^ 1u, 58)));
        if (!ok) break;
        tc_fence_after();
        const uint32_t x = ring + st * Cfg::kStage, ts = tmem + bf * 128u, acc = tmem + Cfg::kAcc;
        mma_weighted<P, 64>(on, acc, ts + 64u, x, i > 0);                                               // dK += ds Q, dQ += ds K
        if (!kind) mma_weighted<P, 64>(on, acc + (uint32_t)P, ts, x + Cfg::kStream / 2, i > 0);         // dV += softmax dOUT
        if (BOTH && i == tiles - 1) {                      // dQ = ds K, over the item's keys
          mma_transposed<P>(on, tmem + Cfg::kAccQ, staged, sheld + (p.held == 2 ? live & 1u : 0u) * Cfg::kHeld);
          commit_if(on, q_free);
        }
        commit_if(on, empty + 8 * st);
        commit_if(on, buf_free + 8 * bf);
        if (i == tiles - 1) {
          commit_if(on, h_empty + 8 * (p.held == 2 ? live & 1u : 0u));
          commit_if(on, acc_full);
        }
        if (++st == (uint32_t)p.stages) st = 0;
        if (++bf == (uint32_t)Cfg::kBuf) { bf = 0; bf_phase ^= 1u; }
      }
      ++live;
    }
  } else {
    // ---------------- element warps ----------------
    const int q = warp & 3, g = (warp - 3) >> 2, rt = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const int reach = p.c.reach, entries = 2 * reach + 1;
    float* group_sums = reinterpret_cast<float*>(gen + (ssums - sheld)) + g * 4 * width;   // with a second set 8 rows behind
    float* sums = group_sums + ((warp - 3) & 3) * width;
    int other_set = p.sets == 2 ? 8 * width : 0;
    const int in_group = ((warp - 3) & 3) * 32 + lane;
    uint32_t n = 0, live = 0, run = 0, st = 0, st_phase = 0, bf = 0, bf_phase = 0;
    bool ok = true, have = false;
    Item prev;
    float below = 0.f, above = 0.f;                    // sums outside the varying part of the bias
    // What undoes the shift of the `n`-th item's score gradients, and of its weights.
    auto unshift = [&](uint32_t n) { return kRelScaled ? power_of_two(-shifts[n & 3u]) : 1.f; };
    auto unshift_weights = [&](uint32_t n) { return kRelScaled ? power_of_two(-max(shifts[n & 3u], 0)) : 1.f; };
    // The `n`-th item's results: dK (group 0) and dV (group 1) of a key, or dQ of a query, 32 features in turn.
    auto store = [&](const Item& it, bool queries, uint32_t acc, bool zero, uint32_t n) {
      const int r = it.t * 128 + rt;
      const Proj& o = queries ? p.dq : g ? p.dv : p.dk;
      sb_half* out = reinterpret_cast<sb_half*>(o.p) + (long long)it.h * o.sH + (long long)it.b * o.sB + (long long)r * o.sR;
      const float f = zero ? 0.f : queries || !g ? p.scale * unshift(n) : unshift_weights(n);
#pragma unroll 1
      for (int c = queries ? g : 0; c < P / 32; c += queries ? 2 : 1) {
        uint32_t v[32];
        if (!zero) {
          tmem_ld32_nowait(acc + lanes + (queries || !g ? 0u : (uint32_t)P) + c * 32, v);
          attn::tmem_ld_wait32(v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        const int rows = queries ? p.c.J : p.c.K;
        if (BOTH && c * 32 < p.c.P)
          store_rows(gen + (sstore - sheld) + (warp - 3) * kStoreBytes, out + c * 32 * o.sP - lane * o.sR, o.sR, o.sP, v, f, min(32, p.c.P - c * 32),
                     rows - r + lane, lane);
        if (!BOTH && r < rows && c * 32 < p.c.P) store_features(out + c * 32 * o.sP, o.sP, v, f, min(32, p.c.P - c * 32));
      }
    };
    auto finish = [&](const Item& it, uint32_t s) {
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full, s & 1u, 59));
      if (!ok) return;
      tc_fence_after();
      store(it, it.kind != 0, tmem + Cfg::kAcc, false, s);
      if (BOTH) store(it, true, tmem + Cfg::kAccQ, false, s);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
    };
    auto add = [&](int rel, float v) {
      if (rel <= -reach) below += v;
      else if (rel >= reach) above += v;
      else sums[rel + reach] += v;
      __syncwarp();
    };
    // a barrier of the group's four warps whose wait is bounded like all others
    uint32_t syncs = 0;
    auto group_sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(g_sync + 8 * g);
      ok = __all_sync(0xffffffffu, mbar_wait(g_sync + 8 * g, syncs & 1u, 61));
      ++syncs;
      return ok;
    };
    // The group's sums of a query tile to memory, to row `place`: 0 for the item's even tiles, 1 for its odd ones, whichever group had
    // them (that depends on the items before).  The rows are left at zero for the next but one such item; with one set it
    // is the next one, and everybody has to be done with them.
    auto flush = [&](const Item& it, int place, float factor) {
      const float lo = warp_sum(below), hi = warp_sum(above);
      below = above = 0.f;
      if (lane == 0) {
        sums[0] = lo;
        sums[2 * reach] = hi;
      }
      if (!group_sync()) return;
      float* out = p.partial + (((long long)it.h * p.c.B * p.nq + (long long)it.b * p.nq + it.t) * 2 + place) * entries;
      for (int i = in_group; i < entries; i += 128) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          v += group_sums[w * width + i];
          group_sums[w * width + i] = 0.f;
        }
        out[i] = v * factor;
      }
      group_sums += other_set;
      sums += other_set;
      other_set = -other_set;
      if (p.sets == 1) group_sync();
    };
    Item w;
    while (ok && take(&w, &ok)) {
      if (w.tiles == 0) {
        store(w, w.kind != 0, 0u, true, 0u);
        if (BOTH) store(w, true, 0u, true, 0u);
        if (BOTH || w.kind) flush(w, g, 1.f);
        continue;
      }
      const int r = w.t * 128 + rt;                    // query or key of this thread
      float lse = INFINITY, dsum = 0.f, weight = 1.f;
      if (w.kind) {
        const uint32_t hb = p.held == 2 ? live & 1u : 0u, hp = p.held == 2 ? live >> 1 : live;
        ok = __all_sync(0xffffffffu, mbar_wait(h_full + 8 * hb, hp & 1u, 60));
        if (!ok) break;
        if (r < p.c.J) {
          const float* rec = reinterpret_cast<const float*>(gen + hb * Cfg::kHeld + 512 * P) + (rt >> 6) * kRecord + (rt & 63);
          lse = rec[0];
          dsum = rec[64];
          weight = rec[128];
        }
      }
      const bool weighted = __any_sync(0xffffffffu, weight != 1.f);
      __syncwarp();
      if (lane == 0) mbar_arrive(h_empty + 8 * (p.held == 2 ? live & 1u : 0u));   // (a group without a tile may come here last)
      bool due = have;                                 // the previous item's results are still to be stored
      // At the first streamed tile of a run, all moving by 64 a tile: relative position of this thread's first column, lowest of
      // the warp's block (its highest is lo + 94), the thread's bound on visible columns and the block's tightest.
      const int step = w.kind ? 64 : -64, moves = w.kind || p.c.causal ? 64 : 0;
      int lim0;
      const int rel0 = w.kind ? -(w.first + r) : r - (w.first + w.t0 * 64);
      if (w.kind) lim0 = p.c.causal ? min(w.keys, w.first + r + 1) : w.keys;
      else lim0 = r < w.keys ? (p.c.causal ? rel0 : -(1 << 30)) : 1 << 30;
      const int lo0 = __shfl_sync(0xffffffffu, rel0, w.kind ? 31 : 0) - (w.kind ? 0 : 63);
      const int tight0 = w.kind ? __reduce_min_sync(0xffffffffu, lim0) : __reduce_max_sync(0xffffffffu, lim0);
      int place = 0;
      for (int done = 0; done < w.tiles && ok; done += w.each) {
        const float* bias = bias_s + (run & 1u) * p.c.pitch;
        ok = __all_sync(0xffffffffu, mbar_wait(b_ready + 8 * (run & 1u), (run >> 1) & 1u, 60));
        if (kRelScaled && w.kind) lse -= (float)shifts[live & 3u];   // (one run)
        // this group's tiles of the run: every second one
        const int skip = (n & 1u) == (uint32_t)g ? 0 : 1;
        place = skip;
        n += w.each;
        auto advance = [&](uint32_t by) {
          st += by;
          if (st >= (uint32_t)p.stages) { st -= p.stages; st_phase ^= 1u; }
          bf += by;
          if (bf >= (uint32_t)Cfg::kBuf) { bf -= Cfg::kBuf; bf_phase ^= 1u; }
        };
        if (skip) advance(1);
        int rel = rel0 + skip * step, lo = lo0 + skip * step, lim = lim0 - skip * moves, tight = tight0 - skip * moves, i = skip;
        if (kRelScaled && !w.kind && shifts[live & 3u] < 0) tight = 1 << 29;   // (score gradients with a factor of their own: masked tiles)
        for (; i < w.each && ok; i += 2) {
          const bool near = lo + 94 > -reach && lo < reach;
          // outside the varying part, a place in the row where the 64 entries in use have the end's value
          const float* bp = bias + (near ? rel + reach + kPad : (lo >= reach ? kPad + 2 * reach : 0) + (w.kind ? 0 : 64));
          const uint32_t ts = tmem + lanes + bf * 128u;
          ok = __all_sync(0xffffffffu, (w.kind || mbar_wait(full + 8 * st, st_phase, 60)) && mbar_wait(s_full + 8 * bf, bf_phase, 60));
          if (!ok) break;
          tc_fence_after();
          if (!BOTH && w.kind) {
            const bool mask = tight < 64;
            if (near || mask || weighted) {
              float up = 0.f, down = 0.f;              // diagonals `lane` and `lane - 32` of a block
              auto block = [&](int c) {
                add(lo + 31 + 32 * c + lane, up);
                add(lo - 1 + 32 * c + lane, down);
                up = down = 0.f;
              };
              auto sum = [&](int e, float ds) {
                const float v = __shfl_sync(0xffffffffu, ds, e - lane);
                if (lane <= e) up += v;
                else down += v;
              };
              auto weigh = [&](int e, float ds) { sum(e, ds * weight); };
              if (mask || weighted) turn_tile<false, true, true>(ts, bp, 0.f, nullptr, nullptr, lse, dsum, lim, p.c.c2, weigh, block);
              else turn_tile<false, true, false>(ts, bp, 0.f, nullptr, nullptr, lse, dsum, lim, p.c.c2, sum, block);
            } else {
              float2 sum = make_float2(0.f, 0.f);
              auto emit = [&](int e, float ds) { (e & 1 ? sum.y : sum.x) += ds; };
              turn_tile<false, false, false>(ts, bp, bp[0], nullptr, nullptr, lse, dsum, lim, p.c.c2, emit, [](int) {});
              (lo >= reach ? above : below) += sum.x + sum.y;
            }
          } else {
            const float* L = reinterpret_cast<const float*>(gen + (ring - sheld) + st * Cfg::kStage + Cfg::kStream);
            auto smaller = [&] { return kRelScaled ? power_of_two(min(shifts[live & 3u], 0)) : 1.f; };
            if (BOTH) {
              // the diagonals of a block run the other way: lane l gets those of key - query = l and l - 32
              float up = 0.f, down = 0.f;
              auto block = [&](int c) {
                add(lo + 63 - 32 * c + lane, up);
                add(lo + 31 - 32 * c + lane, down);
                up = down = 0.f;
              };
              auto sum = [&](int e, float ds) {
                const float v = __shfl_sync(0xffffffffu, ds, e + lane);
                if (lane + e < 32) up += v;
                else down += v;
              };
              const float* W = L + 128;
              int half = 0;
              auto weigh = [&](int e, float ds) { sum(e, ds * W[half + e]); };
              auto next = [&](int c) { block(c); half = 32; };
              const bool some = __any_sync(0xffffffffu, W[lane] != 1.f || W[lane + 32] != 1.f);
              if (live > 0) {                            // the last item's product is done with its score gradients
                ok = __all_sync(0xffffffffu, mbar_wait(q_free, (live - 1u) & 1u, 62));
                if (!ok) break;
              }
              uint8_t* row = gen + (staged - sheld) + i * 16384 + rt * 128;
              if (tight > 0 || some) turn_tile<true, true, true>(ts, bp, 0.f, L, L + 64, 0.f, 0.f, lim, p.c.c2, weigh, next, row, rt & 7, smaller());
              else turn_tile<true, true, false>(ts, bp, 0.f, L, L + 64, 0.f, 0.f, lim, p.c.c2, sum, block, row, rt & 7);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            } else {
              auto none = [](int, float) {};
              auto after = [](int) {};
              if (tight > 0) turn_tile<true, true, true>(ts, bp, 0.f, L, L + 64, 0.f, 0.f, lim, p.c.c2, none, after, nullptr, 0, smaller());
              else if (near) turn_tile<true, true, false>(ts, bp, 0.f, L, L + 64, 0.f, 0.f, lim, p.c.c2, none, after);
              else turn_tile<true, false, false>(ts, bp, bp[0], L, L + 64, 0.f, 0.f, lim, p.c.c2, none, after);
            }
          }
          attn::tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pd_full + 8 * bf);
          if (due) {
            finish(prev, live - 1u);
            if (!ok) break;
            due = false;
          }
          advance(i + 2 <= w.each ? 2 : 1);
          rel += 2 * step;
          lo += 2 * step;
          lim -= 2 * moves;
          tight -= 2 * moves;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(b_empty + 8 * (run & 1u));
        ++run;
      }
      if (!ok) break;
      if (due) {
        finish(prev, live - 1u);
        if (!ok) break;
      }
      if (BOTH || w.kind) flush(w, place, unshift(live));   // (one run, then)
      prev = w;
      have = true;
      ++live;
    }
    if (ok && have) finish(prev, live - 1u);
  }
  flash::drain_after_error();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

}  // namespace rel
