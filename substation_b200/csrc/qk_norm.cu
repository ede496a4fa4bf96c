// Norms of query and key heads and their rotation by position, forward and backward (sb_query_key_norm_rotation and
// sb_backward_query_key_norm_rotation; formulas in the header).  A row is one head of one token.
//
//   forward   y = R(pos) (gain x rs),   rs = (mean x^2 + eps)^(-1/2)
//   backward  g = R(-pos) dy,   dgain = sum g x rs,   dx = rs g gain - x rs^3 mean(g gain x)
//
// A few operations per element: all of it is bound by bytes, each element read once and written once, and for small calls by the
// launch.  Everything is 32 bits between load and store, with one rounding at the end.

#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "ops.h"

namespace sb {

namespace {

constexpr int kDepth = 4;              // rows that a thread of the pieces kernel has on their way
constexpr int kMaxPairs = kNormMaxHead / 2;
constexpr int kMaxPartials = 1184;     // rows of partial sums of a gain's gradient: eight blocks of 148 SMs

// Turns per position of pair i, base^(-2i/rotary) / (2 pi), as a fraction of 2^64: the product with a position, of any sign, wraps
// around as turns do, and its top half is the angle to 2^-32 of a turn however far out the position is.
struct Turns { unsigned long long t[kMaxPairs]; };

struct NormArgs {
  Proj x[2], g[2], y[2];               // queries, keys: input, gradient of the output (backward), result
  const sb_half* gain[2];
  const int* pos;
  long long pos_sB, pos_sJ;
  float* partial[2];                   // backward: a row of P sums per block for the gain's gradient
  int J, tokens, P, rotary, pairing;
  int tile, tiles;                     // tokens of a tile, tiles
  int blocks[2], chunk;                // blocks of queries and of keys; lanes-along-tokens kernel: heads of a block
  float eps;
};

__device__ __forceinline__ float2 cos_sin(int pos, unsigned long long turns_per_position) {
  const unsigned long long t = (unsigned long long)(long long)pos * turns_per_position;
  float s, c;
  sincospif((float)(int)(t >> 32) * 4.656612873077393e-10f, &s, &c);   // halves of a turn: 2^-31
  return make_float2(c, s);
}
struct Place { int b, j; };
__device__ __forceinline__ Place place_of(const NormArgs& a, int token) {
  Place p;
  p.b = token / a.J;
  p.j = token - p.b * a.J;
  return p;
}
__device__ __forceinline__ int position(const NormArgs& a, Place p) { return a.pos[p.b * a.pos_sB + p.j * a.pos_sJ]; }
__device__ __forceinline__ long long token_offset(const Proj& v, Place p) { return p.b * v.sB + p.j * v.sR; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Unit-stride features in 16-byte pieces.  A row belongs to LANES threads with two pieces each, so chosen that both members of
// every pair are in one thread: a row's norm is a few shuffles and its rotation none.  A block takes tiles of tokens, puts
// their angles into shared memory, and its groups of threads walk the query (or key) heads of a token each.  Rows are fetched
// kDepth ahead into a ring that belongs to the thread alone, so that nothing has to be waited for but the copy itself; as
// registers they held half as many bytes in flight.  In the backward pass sum x^2 and sum g gain x are all that a row needs
// from its other threads; the gains' gradients stay in registers until the block's last tile.  Copy bandwidth reached: backward,
// B=4, L=4096, 32 + 8 heads of 128 (503 MB): 104 us, 74 %; forward, B=8, L=512, 16 + 16 heads of 64 (33.6 MB): 9.8 us, 52 %, of
// which about 3 are launch and the first tile's way; a single token for each of 8 samples: 3.7 us.
template <int LANES, bool BWD, bool HALVES>
__global__ void __launch_bounds__(256, 2)
norm_pieces_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Turns turns) {
  constexpr int kGroups = 256 / LANES, kPieces = BWD ? 4 : 2;
  extern __shared__ uint4 smem[];                             // ring [kDepth][kPieces][256], frequencies, angles [2][tile][pairs]
  unsigned long long* freq = reinterpret_cast<unsigned long long*>(smem + kDepth * kPieces * 256);
  float2* cs = reinterpret_cast<float2*>(freq + a.rotary / 2);
  grid_dependency_sync();
  const int pairs = a.rotary / 2, turned = a.rotary / 16, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const uint32_t members = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
  const bool on = lane < a.P / 16, rotates = lane < turned;
  const int f0 = rotates ? 8 * lane : a.rotary + 16 * (lane - turned), f1 = rotates ? f0 + pairs : f0 + 8;
  const int across = kGroups / a.tile, tok = group / across, first_head = group % across;
  const float inv = 1.f / (float)a.P;
  const int w = (int)blockIdx.x < a.blocks[0] ? 0 : 1, mine = (int)blockIdx.x - (w ? a.blocks[0] : 0);
  const Proj &vx = a.x[w], &vg = a.g[w], &vy = a.y[w];
  const int heads = vx.H;
  uint4* slots = smem + threadIdx.x;
  const uint32_t slots_at = (uint32_t)__cvta_generic_to_shared(slots);

  if (!on)                                                    // (what no copy writes stays 0)
    for (int i = 0; i < kDepth * kPieces; ++i) slots[i * 256] = make_uint4(0u, 0u, 0u, 0u);
  const long long x_step = across * vx.sH, g_step = across * vg.sH, y_step = across * vy.sH;

  // the row that is fetched next
  int ft = mine, fh = first_head, fslot = 0;
  const sb_half *fx = nullptr, *fg = nullptr;
  bool flive = false;
  auto at_token = [&] {
    const int token = ft * a.tile + tok;
    flive = on && ft < a.tiles && token < a.tokens && first_head < heads;
    if (flive) {
      const Place p = place_of(a, token);
      fx = reinterpret_cast<const sb_half*>(vx.p) + token_offset(vx, p) + first_head * vx.sH;
      if (BWD) fg = reinterpret_cast<const sb_half*>(vg.p) + token_offset(vg, p) + first_head * vg.sH;
    }
  };
  auto fetch = [&] {
    if (flive) {
      const uint32_t d = slots_at + fslot * kPieces * 4096;
      cp_async16(d, fx + f0);
      cp_async16(d + 4096, fx + f1);
      fx += x_step;
      if (BWD) {
        cp_async16(d + 2 * 4096, fg + f0);
        cp_async16(d + 3 * 4096, fg + f1);
        fg += g_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++fslot == kDepth) fslot = 0;
    fh += across;
    if (fh >= heads) {
      fh = first_head;
      ft += a.blocks[w];
      at_token();
    }
  };
  at_token();
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) fetch();

  float gf[2][8];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int e = 0; e < 8; ++e) gf[x][e] = on ? sb_h2f(a.gain[w][(x ? f1 : f0) + e]) : 0.f;
  for (int i = threadIdx.x; i < pairs; i += 256) freq[i] = turns.t[i];
  __syncthreads();
  float sum[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
  const uint32_t by_pairs = 0xffffffffu / max(pairs, 1) + 1u;   // (i < 2^16: the quotient's high half is exact)
  int slot = 0, buffer = 0;
  for (int t = mine; t < a.tiles; t += a.blocks[w], buffer ^= 1) {
    const int t0 = t * a.tile, token = t0 + tok;
    float2* table = cs + buffer * a.tile * pairs;             // (two in turn: one barrier a tile)
    for (int i = threadIdx.x; i < a.tile * pairs; i += 256) {
      const int k = pairs > 1 ? (int)__umulhi((uint32_t)i, by_pairs) : i;
      if (t0 + k < a.tokens) table[i] = cos_sin(position(a, place_of(a, t0 + k)), freq[i - k * pairs]);
    }
    __syncthreads();
    const bool live = token < a.tokens;
    // halves: the angles of pairs (f0 + e, f1 + e); adjacent: four of the first piece, four of the second
    float2 ang[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      ang[e] = rotates && live ? table[tok * pairs + (HALVES ? f0 + e : (e < 4 ? f0 / 2 + e : f1 / 2 + e - 4))] : make_float2(1.f, 0.f);
    auto turn = [&](float (&u)[8], float (&v)[8], float sign) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float& p = HALVES ? u[e] : (e < 4 ? u[2 * (e & 3)] : v[2 * (e & 3)]);
        float& q = HALVES ? v[e] : (e < 4 ? u[2 * (e & 3) + 1] : v[2 * (e & 3) + 1]);
        const float s = sign * ang[e].y, x = p, y = q;
        p = x * ang[e].x - y * s;
        q = y * ang[e].x + x * s;
      }
    };
    sb_half* py = reinterpret_cast<sb_half*>(vy.p) + (live ? token_offset(vy, place_of(a, token)) : 0) + first_head * vy.sH;
    for (int h = first_head; h < heads; h += across, py += y_step) {
      fetch();
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      const uint4* in = slots + slot * kPieces * 256;
      if (++slot == kDepth) slot = 0;
      if (!live) continue;
      float u[8], v[8], p[8], q[8], sq = 0.f, dot = 0.f;
      unpack8(in[0], u);
      unpack8(in[256], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(u[e], u[e], fmaf(v[e], v[e], sq));
      if (BWD) {
        unpack8(in[512], p);
        unpack8(in[768], q);
        turn(p, q, -1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(p[e] * u[e], gf[0][e], fmaf(q[e] * v[e], gf[1][e], dot));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        sq += __shfl_xor_sync(members, sq, o);
        if (BWD) dot += __shfl_xor_sync(members, dot, o);
      }
      const float rs = rsqrtf(fmaf(sq, inv, a.eps));
      if (!BWD) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[e] *= rs * gf[0][e];
          v[e] *= rs * gf[1][e];
        }
        turn(u, v, 1.f);
      } else {
        const float k = -dot * rs * rs * rs * inv;            // dx = rs g gain - x rs^3 mean(g gain x)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum[e] = fmaf(p[e] * u[e], rs, sum[e]);
          sum[8 + e] = fmaf(q[e] * v[e], rs, sum[8 + e]);
          u[e] = fmaf(p[e] * gf[0][e], rs, u[e] * k);
          v[e] = fmaf(q[e] * gf[1][e], rs, v[e] * k);
        }
      }
      if (on) {
        *reinterpret_cast<uint4*>(py + f0) = pack8(u);
        *reinterpret_cast<uint4*>(py + f1) = pack8(v);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (BWD) {
    // the block's sums: over a warp's groups by shuffles, over the warps in shared memory
    float* part = reinterpret_cast<float*>(smem);             // [8][P]
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = sum[e];
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if ((threadIdx.x & 31) < LANES && on) part[(threadIdx.x >> 5) * a.P + (e < 8 ? f0 : f1 - 8) + e] = v;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < a.P; p += 256) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += part[i * a.P + p];
      a.partial[w][(long long)mine * a.P + p] = v;
    }
  }
}

// Any strides, any head size, lanes along tokens (what head-first projections have side by side).  Warp w of a block has the
// pairs w, w + WARPS, .. of features (rotary pairs, then neighbours), SLOTS at most, of TOKENS tokens per lane, and keeps their
// angles in registers while the block walks its heads; a row's sums go through shared memory.  The next head's elements are on
// their way meanwhile, as long as registers last.  TOKENS = 2: tokens side by side in memory, in 32-bit words.  Off: the type that
// holds a feature's offset, 32 bits wherever a head's features span less than 2^31 elements (64-bit products of strides were most
// of the instructions).  Forward, B=12, L=200, 12 + 12 heads of 64, head-first (14.7 MB): 8.2 us, 27 % of the copy bandwidth, one wave
// of blocks that are chains of as many heads as each has (11.9 us with single tokens, eight heads a block, no head on its way).
template <int TOKENS> struct Elements;                        // of one feature: TOKENS tokens
template <> struct Elements<1> {
  sb_half h;
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = sb_h2f(h); }
  __device__ __forceinline__ static Elements of(const float (&v)[1]) { return {sb_f2h(v[0])}; }
};
template <> struct Elements<2> {
  sb_half2 h;
  __device__ __forceinline__ void get(float (&v)[2]) const {
    const float2 f = sb_h22f2(h);
    v[0] = f.x;
    v[1] = f.y;
  }
  __device__ __forceinline__ static Elements of(const float (&v)[2]) { return {sb_f2h2(v[0], v[1])}; }
};
template <int WARPS, int SLOTS, int TOKENS, bool BWD, class Off>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
norm_strided_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Turns turns) {
  using El = Elements<TOKENS>;
  constexpr bool kAhead = SLOTS <= 4 && !(BWD && TOKENS == 2);   // (no registers left there: 19.2 us with, 18.4 without)
  __shared__ float2 part[2][WARPS][32 * TOKENS];
  grid_dependency_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = a.rotary / 2, slots = (a.P + 1) / 2;
  const int w = (int)blockIdx.x < a.blocks[0] ? 0 : 1, mine = (int)blockIdx.x - (w ? a.blocks[0] : 0);
  const int chunks = (a.x[w].H + a.chunk - 1) / a.chunk, stride = a.blocks[w] / chunks;
  const int h_from = mine % chunks * a.chunk, h_to = min(a.x[w].H, h_from + a.chunk);
  const float inv = 1.f / (float)a.P;
  // the two features of each slot: place in x, g and y (of the first where there is none), gain (then 0)
  Off xo[SLOTS][2], go[SLOTS][2], yo[SLOTS][2];
  float gain[SLOTS][2], sum[SLOTS][2];
  uint32_t there = 0;
  auto feature = [&](int i, int e) {
    const int u = warp + WARPS * i;
    return u < pairs && a.pairing == SB_PAIR_HALVES ? u + e * pairs : 2 * u + e;
  };
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool is = warp + WARPS * i < slots && feature(i, e) < a.P;
      const int f = is ? feature(i, e) : 0;
      there |= (is ? 1u : 0u) << (2 * i + e);
      gain[i][e] = is ? sb_h2f(a.gain[w][f]) : 0.f;
      xo[i][e] = (Off)(f * a.x[w].sP);
      go[i][e] = BWD ? (Off)(f * a.g[w].sP) : 0;
      yo[i][e] = (Off)(f * a.y[w].sP);
      sum[i][e] = 0.f;
    }
  }
  int turnstile = 0;
  for (int t = mine / chunks; t < a.tiles; t += stride) {
    const int token = (t * 32 + lane) * TOKENS;               // (two of them are of one sample and both there, or neither)
    const bool live = token < a.tokens;
    const Place at = place_of(a, live ? token : 0);
    const sb_half* X = reinterpret_cast<const sb_half*>(a.x[w].p) + token_offset(a.x[w], at) + h_from * a.x[w].sH;
    const sb_half* G = BWD ? reinterpret_cast<const sb_half*>(a.g[w].p) + token_offset(a.g[w], at) + h_from * a.g[w].sH : nullptr;
    sb_half* Y = reinterpret_cast<sb_half*>(a.y[w].p) + token_offset(a.y[w], at) + h_from * a.y[w].sH;
    El x[SLOTS][2], g[SLOTS][2], x_next[SLOTS][2], g_next[SLOTS][2];
    auto load = [&](El (&lx)[SLOTS][2], El (&lg)[SLOTS][2]) { // (a feature that is not there reads the first and counts 0)
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          lx[i][e] = *reinterpret_cast<const El*>(X + xo[i][e]);
          if (BWD) lg[i][e] = *reinterpret_cast<const El*>(G + go[i][e]);
        }
      X += a.x[w].sH;
      if (BWD) G += a.g[w].sH;
    };
    if (kAhead) load(x_next, g_next);
    float2 ang[SLOTS][TOKENS];
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
      const int pos = position(a, Place{at.b, at.j + (live ? k : 0)});
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) ang[i][k] = warp + WARPS * i < pairs ? cos_sin(pos, turns.t[warp + WARPS * i]) : make_float2(1.f, 0.f);
    }
    // features (2 of a slot, of all tokens) as numbers, and gradients turned back
    auto numbers = [&](int i, float (&u)[TOKENS], float (&v)[TOKENS], float (&p)[TOKENS], float (&q)[TOKENS]) {
      x[i][0].get(u);
      x[i][1].get(v);
      if (BWD) {
        g[i][0].get(p);
        g[i][1].get(q);
      }
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        if (!((there >> (2 * i)) & 1u)) u[k] = p[k] = 0.f;
        if (!((there >> (2 * i + 1)) & 1u)) v[k] = q[k] = 0.f;
        if (BWD) {
          const float c = ang[i][k].x, s = ang[i][k].y, y = p[k], z = q[k];
          p[k] = y * c + z * s;
          q[k] = z * c - y * s;
        }
      }
    };
#pragma unroll 1
    for (int h = h_from; h < h_to; ++h, turnstile ^= 1, Y += a.y[w].sH) {
      if (kAhead) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[i][e] = x_next[i][e];
            if (BWD) g[i][e] = g_next[i][e];
          }
        if (h + 1 < h_to) load(x_next, g_next);
      } else {
        load(x, g);
      }
      float sq[TOKENS], dot[TOKENS];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) sq[k] = dot[k] = 0.f;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        float u[TOKENS], v[TOKENS], p[TOKENS], q[TOKENS];
        numbers(i, u, v, p, q);
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
          sq[k] = fmaf(u[k], u[k], fmaf(v[k], v[k], sq[k]));
          if (BWD) dot[k] = fmaf(p[k] * gain[i][0], u[k], fmaf(q[k] * gain[i][1], v[k], dot[k]));
        }
      }
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) part[turnstile][warp][lane * TOKENS + k] = make_float2(sq[k], dot[k]);
      __syncthreads();
      float rs[TOKENS], mean[TOKENS];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        sq[k] = dot[k] = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
          const float2 s = part[turnstile][i][lane * TOKENS + k];
          sq[k] += s.x;
          if (BWD) dot[k] += s.y;
        }
        rs[k] = rsqrtf(fmaf(sq[k], inv, a.eps));
        mean[k] = dot[k] * rs[k] * inv;
      }
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        float u[TOKENS], v[TOKENS], p[TOKENS], q[TOKENS];
        numbers(i, u, v, p, q);
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
          u[k] *= rs[k];
          v[k] *= rs[k];
          if (!BWD) {
            const float c = ang[i][k].x, s = ang[i][k].y, y = u[k] * gain[i][0], z = v[k] * gain[i][1];
            u[k] = y * c - z * s;
            v[k] = z * c + y * s;
          } else {
            if (live) {                                       // (what lies behind the last token is token 0 again)
              sum[i][0] = fmaf(p[k], u[k], sum[i][0]);
              sum[i][1] = fmaf(q[k], v[k], sum[i][1]);
            }
            u[k] = rs[k] * (p[k] * gain[i][0] - u[k] * mean[k]);
            v[k] = rs[k] * (q[k] * gain[i][1] - v[k] * mean[k]);
          }
        }
        if (live && ((there >> (2 * i)) & 1u)) *reinterpret_cast<El*>(Y + yo[i][0]) = El::of(u);
        if (live && ((there >> (2 * i + 1)) & 1u)) *reinterpret_cast<El*>(Y + yo[i][1]) = El::of(v);
      }
    }
  }
#pragma unroll
  for (int i = 0; BWD && i < SLOTS; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = warp_sum(sum[i][e]);
      if (lane == 0 && ((there >> (2 * i + e)) & 1u)) a.partial[w][(long long)mine * a.P + feature(i, e)] = v;
    }
}

// Features side by side, but off the 16-byte grid or with pairs that pieces do not hold: a warp per row, a lane per pair (SLOTS of them,
// 32 apart), kRows heads of a token at a time, whose elements are all asked for before any is used.  Angles stay for a token's heads.
// Bound by the 64 bytes of its loads: B=8, L=512, 16 + 16 heads of 64, one element off the grid: 24.6 us (pieces on the grid 9.8; lanes
// along tokens 113, each of which touches 32 rows with a load).
template <int SLOTS, bool BWD>
__global__ void __launch_bounds__(256, 2)
norm_rows_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Turns turns) {
  constexpr int kRows = SLOTS == 1 ? 4 : SLOTS == 2 ? 2 : 1;
  __shared__ float part[BWD ? 8 * kNormMaxHead : 1];
  grid_dependency_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = a.rotary / 2, slots = (a.P + 1) / 2;
  const int w = (int)blockIdx.x < a.blocks[0] ? 0 : 1, mine = (int)blockIdx.x - (w ? a.blocks[0] : 0), heads = a.x[w].H;
  const float inv = 1.f / (float)a.P;
  int f[SLOTS][2];                                            // -1: not there
  float gain[SLOTS][2], sum[SLOTS][2];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int u = lane + 32 * i, n = u < pairs && a.pairing == SB_PAIR_HALVES ? u + e * pairs : 2 * u + e;
      f[i][e] = u < slots && n < a.P ? n : -1;
      gain[i][e] = f[i][e] >= 0 ? sb_h2f(a.gain[w][f[i][e]]) : 0.f;
      sum[i][e] = 0.f;
    }
  for (int token = mine * 8 + warp; token < a.tokens; token += a.blocks[w] * 8) {
    const Place at = place_of(a, token);
    const sb_half* X = reinterpret_cast<const sb_half*>(a.x[w].p) + token_offset(a.x[w], at);
    const sb_half* G = BWD ? reinterpret_cast<const sb_half*>(a.g[w].p) + token_offset(a.g[w], at) : nullptr;
    sb_half* Y = reinterpret_cast<sb_half*>(a.y[w].p) + token_offset(a.y[w], at);
    const int pos = position(a, at);
    float2 ang[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) ang[i] = lane + 32 * i < pairs ? cos_sin(pos, turns.t[lane + 32 * i]) : make_float2(1.f, 0.f);
    for (int h0 = 0; h0 < heads; h0 += kRows) {
      float x[kRows][SLOTS][2], g[kRows][SLOTS][2];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool is = f[i][e] >= 0 && h0 + r < heads;
            x[r][i][e] = is ? sb_h2f(X[(h0 + r) * a.x[w].sH + f[i][e]]) : 0.f;
            if (BWD) g[r][i][e] = is ? sb_h2f(G[(h0 + r) * a.g[w].sH + f[i][e]]) : 0.f;
          }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
          const float u = x[r][i][0], v = x[r][i][1];
          sq = fmaf(u, u, fmaf(v, v, sq));
          if (BWD) {
            const float c = ang[i].x, s = ang[i].y, p = g[r][i][0], q = g[r][i][1];
            g[r][i][0] = p * c + q * s;                       // turned back
            g[r][i][1] = q * c - p * s;
            dot = fmaf(g[r][i][0] * gain[i][0], u, fmaf(g[r][i][1] * gain[i][1], v, dot));
          }
        }
        sq = group_sum<32>(sq);
        if (BWD) dot = group_sum<32>(dot);
        const float rs = rsqrtf(fmaf(sq, inv, a.eps)), mean = BWD ? dot * rs * inv : 0.f;
        if (h0 + r >= heads) continue;                        // (the same for the whole warp)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
          float u = x[r][i][0] * rs, v = x[r][i][1] * rs;
          if (!BWD) {
            const float c = ang[i].x, s = ang[i].y, p = u * gain[i][0], q = v * gain[i][1];
            u = p * c - q * s;
            v = q * c + p * s;
          } else {
            const float p = g[r][i][0], q = g[r][i][1];
            sum[i][0] = fmaf(p, u, sum[i][0]);
            sum[i][1] = fmaf(q, v, sum[i][1]);
            u = rs * (p * gain[i][0] - u * mean);
            v = rs * (q * gain[i][1] - v * mean);
          }
          if (f[i][0] >= 0) Y[(h0 + r) * a.y[w].sH + f[i][0]] = sb_f2h(u);
          if (f[i][1] >= 0) Y[(h0 + r) * a.y[w].sH + f[i][1]] = sb_f2h(v);
        }
      }
    }
  }
  if (BWD) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (f[i][e] >= 0) part[warp * a.P + f[i][e]] = sum[i][e];
    __syncthreads();
    for (int p = threadIdx.x; p < a.P; p += 256) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += part[i * a.P + p];
      a.partial[w][(long long)mine * a.P + p] = v;
    }
  }
}

// out[p] = sum of the blocks' rows in a fixed order: 32 threads a column take every 32nd row, then a tree.  Latency alone: 2.9 us for
// 296 rows of 64.
__global__ void __launch_bounds__(1024)
gain_finish_kernel(const float* q_partial, const float* k_partial, int q_rows, int k_rows, int P, sb_half* q, sb_half* k) {
  __shared__ float part[32][33];
  grid_dependency_sync();
  const float* partial = blockIdx.y ? k_partial : q_partial;
  const int rows = blockIdx.y ? k_rows : q_rows, p = blockIdx.x * 32 + (threadIdx.x & 31), i = threadIdx.x >> 5;
  float s = 0.f;
  if (p < P)
#pragma unroll 8
    for (int b = i; b < rows; b += 32) s += partial[(long long)b * P + p];
  part[i][threadIdx.x & 31] = s;
  __syncthreads();
  s = warp_sum(part[threadIdx.x & 31][i]);                    // warp i: column i
  if ((threadIdx.x & 31) == 0 && blockIdx.x * 32 + i < P) (blockIdx.y ? k : q)[blockIdx.x * 32 + i] = sb_f2h(s);
}

// The frequencies of a rotation.  Each takes about 0.3 us of host time to work out, so a thread keeps those of the last eight rotations: a
// model's layers may alternate between a few.
const Turns& turns_of(const Rotation& r) {
  struct Known {
    Turns turns;
    double base = 0.0;
    int rotary = -1;
  };
  static thread_local Known known[8];
  static thread_local int next = 0;
  for (const Known& k : known)
    if (k.base == r.base && k.rotary == r.rotary) return k.turns;
  Known& k = known[next];
  next = (next + 1) % 8;
  for (int i = 0; i < kMaxPairs; ++i) {
    k.turns.t[i] = 0;
    if (2 * i >= r.rotary) continue;
    const long double turns = std::pow((long double)r.base, -2.0L * i / r.rotary) / 6.283185307179586476925286766559L;
    const long double scaled = std::ldexp(turns - std::floor(turns), 64);
    k.turns.t[i] = scaled < 18446744073709551615.0L ? (unsigned long long)scaled : ~0ull;
  }
  k.base = r.base;
  k.rotary = r.rotary;
  return k.turns;
}

NormArgs norm_args(const Proj& q, const Proj& k, const void* q_gain, const void* k_gain, const View2& pos, const Rotation& rot) {
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.x[0] = q; a.x[1] = k;
  a.gain[0] = reinterpret_cast<const sb_half*>(q_gain);
  a.gain[1] = reinterpret_cast<const sb_half*>(k_gain);
  a.pos = reinterpret_cast<const int*>(pos.p); a.pos_sB = pos.sB; a.pos_sJ = pos.sJ;
  a.J = q.R; a.tokens = q.B * q.R; a.P = q.P;
  a.rotary = rot.rotary; a.pairing = rot.pairing; a.eps = rot.eps;
  return a;
}

// Unit-stride features in 16-byte pieces that both members of a pair are two of.
bool in_pieces(const Proj& v, int rotary) {
  auto ok = [](long long n, long long stride) { return n == 1 || stride % 8 == 0; };
  return v.H == 0 || (v.sP == 1 && v.P % 16 == 0 && rotary % 16 == 0 && ok(v.H, v.sH) && ok(v.B, v.sB) && ok(v.R, v.sR) &&
                      !(reinterpret_cast<uintptr_t>(v.p) & 15u));
}

template <int LANES, bool BWD>
int launch_pieces(cudaStream_t s, NormArgs& a, const Rotation& rot, int* rows) {
  // Four groups of threads a token, so that one has several heads to fetch at a time; fewer tokens a block where that leaves SMs
  // without one (single tokens).
  const int sms = usable_sms(device_facts().sms), groups = 256 / LANES;
  for (a.tile = groups / 4; a.tile > 1 && (a.tokens + a.tile - 1) / a.tile < sms; a.tile /= 2) {}
  a.tiles = (a.tokens + a.tile - 1) / a.tile;
  // Two blocks an SM at a time; the backward pass has room for the sums of so many.  A tile costs its heads and, for angles and
  // barriers, about as much as six more, and so queries and keys share the blocks.
  const int most = std::min(2 * sms, kMaxPartials), cost[2] = {a.x[0].H + 6, a.x[1].H > 0 ? a.x[1].H + 6 : 0};
  for (int w = 0; w < 2; ++w)
    a.blocks[w] = rows[w] = cost[w] ? std::min(a.tiles, std::max(1, (most * cost[w] + (w ? cost[0] + cost[1] - 1 : 0)) / (cost[0] + cost[1]))) : 0;
  const size_t smem = kDepth * (BWD ? 4 : 2) * 4096 + sizeof(unsigned long long) * (a.rotary / 2) + 2 * sizeof(float2) * a.tile * (a.rotary / 2);
  auto kernel = a.pairing == SB_PAIR_HALVES ? norm_pieces_kernel<LANES, BWD, true> : norm_pieces_kernel<LANES, BWD, false>;
  SB_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), 100 * 1024));
  SB_LAUNCH_OK(launch_k(kernel, a.blocks[0] + a.blocks[1], 256, smem, s, a, turns_of(rot)));
  return SB_OK;
}
template <int SLOTS, bool BWD>
int launch_rows(cudaStream_t s, NormArgs& a, const Rotation& rot, int* rows) {
  a.tiles = (a.tokens + 7) / 8;
  const long long most = std::min(4 * usable_sms(device_facts().sms), kMaxPartials), heads = a.x[0].H + a.x[1].H;
  for (int w = 0; w < 2; ++w)    // queries and keys share the blocks by their heads
    a.blocks[w] = rows[w] = a.x[w].H ? (int)std::min<long long>(a.tiles, std::max(1ll, most * a.x[w].H / heads)) : 0;
  SB_LAUNCH_OK(launch_k(norm_rows_kernel<SLOTS, BWD>, a.blocks[0] + a.blocks[1], 256, 0, s, a, turns_of(rot)));
  return SB_OK;
}
template <int WARPS, int SLOTS, int TOKENS, bool BWD>
int launch_strided(cudaStream_t s, NormArgs& a, const Rotation& rot, int* rows) {
  const int resident = 16 / WARPS * usable_sms(device_facts().sms);
  a.tiles = (a.tokens + 32 * TOKENS - 1) / (32 * TOKENS);
  // Up to eight heads a block, which share its angles and everything else that a block begins with, about as much as two more
  // heads; what matters is how often the SMs are filled with blocks.
  long long least = 0;
  for (int c = 8; c >= 1; --c) {
    const long long blocks = (long long)a.tiles * ((a.x[0].H + c - 1) / c + (a.x[1].H + c - 1) / c), cost = (blocks + resident - 1) / resident * (c + 2);
    if (c == 8 || cost < least) {
      least = cost;
      a.chunk = c;
    }
  }
  if (BWD) a.chunk = std::max({a.chunk, (a.x[0].H + kMaxPartials - 1) / kMaxPartials, (a.x[1].H + kMaxPartials - 1) / kMaxPartials});
  for (int w = 0; w < 2; ++w) {
    const int chunks = (a.x[w].H + a.chunk - 1) / a.chunk;
    // (every chunk has the same number of blocks; the backward pass bounds their number by its rows of sums)
    const int each = BWD && chunks > 0 ? std::min(a.tiles, kMaxPartials / chunks) : a.tiles;
    a.blocks[w] = rows[w] = chunks * each;
  }
  bool narrow = true;
  for (int w = 0; w < 2; ++w)
    for (const Proj* v : {&a.x[w], &a.y[w], &a.g[w]}) narrow = narrow && std::llabs(v->sP) < (1ll << 31) / kNormMaxHead;
  auto kernel = narrow ? norm_strided_kernel<WARPS, SLOTS, TOKENS, BWD, int> : norm_strided_kernel<WARPS, SLOTS, TOKENS, BWD, long long>;
  SB_LAUNCH_OK(launch_k(kernel, a.blocks[0] + a.blocks[1], 32 * WARPS, 0, s, a, turns_of(rot)));
  return SB_OK;
}
template <bool BWD>
int launch_norm(cudaStream_t s, NormArgs& a, const Rotation& rot, int* rows) {
  bool pieces = true;
  for (int w = 0; w < 2; ++w)
    for (const Proj* v : {&a.x[w], &a.y[w], &a.g[w]}) pieces = pieces && (v->p == nullptr || in_pieces(*v, a.rotary));
  if (pieces) {
    if (a.P <= 16) return launch_pieces<1, BWD>(s, a, rot, rows);
    if (a.P <= 32) return launch_pieces<2, BWD>(s, a, rot, rows);
    if (a.P <= 64) return launch_pieces<4, BWD>(s, a, rot, rows);
    if (a.P <= 128) return launch_pieces<8, BWD>(s, a, rot, rows);
    return launch_pieces<16, BWD>(s, a, rot, rows);
  }
  // features side by side
  bool side = true;
  for (int w = 0; w < 2; ++w)
    for (const Proj* v : {&a.x[w], &a.y[w], &a.g[w]}) side = side && (v->p == nullptr || v->sP == 1);
  if (side) return a.P <= 64 ? launch_rows<1, BWD>(s, a, rot, rows) : a.P <= 128 ? launch_rows<2, BWD>(s, a, rot, rows) : launch_rows<4, BWD>(s, a, rot, rows);
  // tokens in twos where they lie side by side in 32-bit words
  bool twos = a.J % 2 == 0;
  for (int w = 0; w < 2; ++w)
    for (const Proj* v : {&a.x[w], &a.y[w], &a.g[w]})
      twos = twos && (v->p == nullptr || (v->sR == 1 && !((v->sP | v->sH | v->sB) & 1) && !(reinterpret_cast<uintptr_t>(v->p) & 3u)));
  if (a.P <= 64) return twos ? launch_strided<8, 4, 2, BWD>(s, a, rot, rows) : launch_strided<8, 4, 1, BWD>(s, a, rot, rows);
  if (a.P <= 128) return twos ? launch_strided<16, 4, 2, BWD>(s, a, rot, rows) : launch_strided<16, 4, 1, BWD>(s, a, rot, rows);
  return launch_strided<16, 8, 1, BWD>(s, a, rot, rows);
}

}  // namespace

size_t qk_norm_scratch_bytes() { return sizeof(float) * 2 * kNormMaxHead * kMaxPartials; }

int launch_qk_norm_fwd(cudaStream_t s, Proj q, Proj k, const void* q_gain, const void* k_gain, View2 pos, Proj q_out, Proj k_out,
                       const Rotation& rot) {
  NormArgs a = norm_args(q, k, q_gain, k_gain, pos, rot);
  if (a.tokens == 0) return SB_OK;
  a.y[0] = q_out; a.y[1] = k_out;
  int rows[2];
  return launch_norm<false>(s, a, rot, rows);
}

int launch_qk_norm_bwd(cudaStream_t s, void* scratch, Proj dq_out, Proj dk_out, Proj q, Proj k, const void* q_gain, const void* k_gain,
                       View2 pos, Proj dq, Proj dk, void* dq_gain, void* dk_gain, const Rotation& rot) {
  NormArgs a = norm_args(q, k, q_gain, k_gain, pos, rot);
  a.g[0] = dq_out; a.g[1] = dk_out;
  a.y[0] = dq; a.y[1] = dk;
  a.partial[0] = reinterpret_cast<float*>(scratch);
  a.partial[1] = a.partial[0] + kMaxPartials * kNormMaxHead;
  int rows[2] = {0, 0};                  // without tokens the gains' gradients are 0
  if (a.tokens > 0) SB_TRY(launch_norm<true>(s, a, rot, rows));
  SB_LAUNCH_OK(launch_k(gain_finish_kernel, dim3((a.P + 31) / 32, k.H > 0 ? 2 : 1), 1024, 0, s, a.partial[0], a.partial[1], rows[0], rows[1], a.P,
                        reinterpret_cast<sb_half*>(dq_gain), reinterpret_cast<sb_half*>(dk_gain)));
  return SB_OK;
}

}  // namespace sb
