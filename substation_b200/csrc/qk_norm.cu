// Norms of query and key heads and their rotation by position, forward and backward (sb_query_key_norm_rotation and
// sb_backward_query_key_norm_rotation; formulas in the header).  A row is one head of one token.

#include <algorithm>
#include <cmath>

#include "ops.h"

namespace sb {

namespace {

constexpr int kTokens = 32;            // tokens of a block of the tile kernels
constexpr int kMaxPairs = kNormMaxHead / 2;
constexpr int kMaxPartials = 1184;     // rows of partial sums of the gains' gradients: eight blocks of 148 SMs

// Turns per position of pair i: base^(-2i/rotary) / (2 pi).  Angles are counted in turns and reduced to a fraction of one in
// 64 bits: a position of 2^31 then still has 22 bits behind the binary point.
struct Turns { double t[kMaxPairs]; };

struct NormArgs {
  Proj x[2], g[2], y[2];               // queries, keys: input, gradient of the output (backward), result
  const sb_half* gain[2];
  const int* pos;
  long long pos_sB, pos_sJ;
  float* partial;                      // backward: [blocks of tokens][2][P]
  int J, tokens, P, rotary, pairing;
  int vary_tokens[2][3];               // the tile kernels' lanes run along tokens (x, g, y)
  float eps;
};

__device__ __forceinline__ float2 cos_sin(int pos, double turns_per_position) {
  const double t = (double)pos * turns_per_position;
  float s, c;
  sincospif(2.f * (float)(t - rint(t)), &s, &c);
  return make_float2(c, s);
}

__device__ __forceinline__ long long row_offset(const Proj& v, int token, int J, int h) {
  return (long long)(token / J) * v.sB + (long long)(token % J) * v.sR + (long long)h * v.sH;
}

// tile[t][p] = v[p, h, tokens t0 ...], lanes along tokens or along features, whichever is nearer in memory
__device__ __forceinline__ void load_rows(float* tile, int pitch, const Proj& v, const NormArgs& a, int t0, int h, bool along_tokens) {
  const sb_half* base = reinterpret_cast<const sb_half*>(v.p);
  const int n = min(kTokens, a.tokens - t0);
  if (along_tokens) {
    const int t = threadIdx.x & 31;
    if (t < n) {
      const long long o = row_offset(v, t0 + t, a.J, h);
      for (int p = threadIdx.x >> 5; p < a.P; p += 8) tile[t * pitch + p] = sb_h2f(base[o + (long long)p * v.sP]);
    }
  } else {
    for (int t = threadIdx.x >> 5; t < n; t += 8) {
      const long long o = row_offset(v, t0 + t, a.J, h);
      for (int p = threadIdx.x & 31; p < a.P; p += 32) tile[t * pitch + p] = sb_h2f(base[o + (long long)p * v.sP]);
    }
  }
}
__device__ __forceinline__ void store_rows(const float* tile, int pitch, const Proj& v, const NormArgs& a, int t0, int h, bool along_tokens) {
  sb_half* base = reinterpret_cast<sb_half*>(v.p);
  const int n = min(kTokens, a.tokens - t0);
  if (along_tokens) {
    const int t = threadIdx.x & 31;
    if (t < n) {
      const long long o = row_offset(v, t0 + t, a.J, h);
      for (int p = threadIdx.x >> 5; p < a.P; p += 8) base[o + (long long)p * v.sP] = sb_f2h(tile[t * pitch + p]);
    }
  } else {
    for (int t = threadIdx.x >> 5; t < n; t += 8) {
      const long long o = row_offset(v, t0 + t, a.J, h);
      for (int p = threadIdx.x & 31; p < a.P; p += 32) base[o + (long long)p * v.sP] = sb_f2h(tile[t * pitch + p]);
    }
  }
}

// Any strides, any head size: a block takes 32 tokens, keeps their angles in shared memory and walks the heads; eight threads
// a row.  Forward and backward (BWD), queries and keys one after the other.
template <bool BWD>
__global__ void __launch_bounds__(256)
norm_tile_kernel(const NormArgs a, const Turns turns) {
  extern __shared__ float smem[];
  const int pairs = a.rotary / 2, pitch = a.P | 1;
  float* tx = smem;                                 // [kTokens][pitch]
  float* tg = tx + kTokens * pitch;                 // the same, backward only
  float2* cs = reinterpret_cast<float2*>(smem + (((BWD ? 2 : 1) * kTokens * pitch + 1) & ~1));
  grid_dependency_sync();
  const int part = threadIdx.x & 7, t = threadIdx.x >> 3;
  const float inv = 1.f / (float)a.P;
  for (int which = 0; which < 2; ++which)
    if (BWD && a.x[which].H > 0)
      for (int p = threadIdx.x; p < a.P; p += 256) a.partial[((long long)blockIdx.x * 2 + which) * a.P + p] = 0.f;
  for (int t0 = blockIdx.x * kTokens; t0 < a.tokens; t0 += gridDim.x * kTokens) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTokens * pairs; i += 256) {
      const int tt = t0 + i / pairs;
      cs[i] = tt < a.tokens ? cos_sin(a.pos[(long long)(tt / a.J) * a.pos_sB + (long long)(tt % a.J) * a.pos_sJ], turns.t[i % pairs])
                            : make_float2(1.f, 0.f);
    }
    for (int which = 0; which < 2; ++which) {
      const Proj& vx = a.x[which];
      for (int h = 0; h < vx.H; ++h) {
        __syncthreads();
        load_rows(tx, pitch, vx, a, t0, h, a.vary_tokens[which][0]);
        if (BWD) load_rows(tg, pitch, a.g[which], a, t0, h, a.vary_tokens[which][1]);
        __syncthreads();
        const bool row = t0 + t < a.tokens;
        float* x = tx + t * pitch;
        float* g = tg + t * pitch;
        float sum = 0.f;
        if (row)
          for (int p = part; p < a.P; p += 8) sum = fmaf(x[p], x[p], sum);
        const float r = rsqrtf(group_sum<8>(sum) * inv + a.eps);
        auto pair = [&](int i, int* p, int* q) {
          if (a.pairing == SB_PAIR_HALVES) { *p = i; *q = i + pairs; }
          else { *p = 2 * i; *q = 2 * i + 1; }
        };
        const sb_half* gain = a.gain[which];
        if (!BWD) {
          if (row) {
            for (int i = part; i < pairs; i += 8) {
              int p, q;
              pair(i, &p, &q);
              const float2 w = cs[t * pairs + i];
              const float u = x[p] * r * sb_h2f(gain[p]), v = x[q] * r * sb_h2f(gain[q]);
              x[p] = u * w.x - v * w.y;
              x[q] = v * w.x + u * w.y;
            }
            for (int p = a.rotary + part; p < a.P; p += 8) x[p] = x[p] * r * sb_h2f(gain[p]);
          }
        } else {
          // g turned back; x becomes n
          float dot = 0.f;
          if (row) {
            for (int i = part; i < pairs; i += 8) {
              int p, q;
              pair(i, &p, &q);
              const float2 w = cs[t * pairs + i];
              const float u = g[p], v = g[q];
              g[p] = u * w.x + v * w.y;
              g[q] = v * w.x - u * w.y;
              x[p] *= r;
              x[q] *= r;
              dot += g[p] * sb_h2f(gain[p]) * x[p] + g[q] * sb_h2f(gain[q]) * x[q];
            }
            for (int p = a.rotary + part; p < a.P; p += 8) {
              x[p] *= r;
              dot += g[p] * sb_h2f(gain[p]) * x[p];
            }
          }
          const float mean = group_sum<8>(dot) * inv;
          __syncthreads();
          const int n = min(kTokens, a.tokens - t0);
          for (int p = threadIdx.x; p < a.P; p += 256) {
            float s = 0.f;
            for (int k = 0; k < n; ++k) s = fmaf(tg[k * pitch + p], tx[k * pitch + p], s);
            a.partial[((long long)blockIdx.x * 2 + which) * a.P + p] += s;
          }
          __syncthreads();
          if (row)
            for (int p = part; p < a.P; p += 8) x[p] = r * (g[p] * sb_h2f(gain[p]) - x[p] * mean);
        }
        __syncthreads();
        store_rows(tx, pitch, a.y[which], a, t0, h, a.vary_tokens[which][2]);
      }
    }
  }
}

// out[which][p] = sum of the blocks' partial sums in a fixed order: 16 threads a column take every 16th row, then a tree.
__global__ void __launch_bounds__(512)
gain_finish_kernel(const float* __restrict__ partial, int blocks, int P, sb_half* q, sb_half* k) {
  __shared__ float part[16][33];
  grid_dependency_sync();
  const int which = blockIdx.y, p = blockIdx.x * 32 + (threadIdx.x & 31), i = threadIdx.x >> 5;
  float s = 0.f;
  if (p < P)
    for (int b = i; b < blocks; b += 16) s += partial[((long long)b * 2 + which) * P + p];
  part[i][threadIdx.x & 31] = s;
  __syncthreads();
  if (i == 0 && p < P) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = part[j][threadIdx.x & 31];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int j = 0; j < o; ++j) v[j] += v[j + o];
    (which ? k : q)[p] = sb_f2h(v[0]);
  }
}

// The frequencies of one rotation, remembered per thread: a program uses one or two.
const Turns& turns_of(const Rotation& r) {
  static thread_local Turns t;
  static thread_local double base = 0.0;
  static thread_local int rotary = -1;
  if (base != r.base || rotary != r.rotary) {
    for (int i = 0; i < kMaxPairs; ++i)
      t.t[i] = 2 * i < r.rotary ? std::pow(r.base, -2.0 * i / r.rotary) / 6.283185307179586476925286766559 : 0.0;
    base = r.base;
    rotary = r.rotary;
  }
  return t;
}

bool along_tokens(const Proj& v) {
  auto mag = [](long long s) { return s < 0 ? -s : s; };
  return v.R > 1 && mag(v.sR) < mag(v.sP);
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

template <bool BWD>
int launch_tiles(cudaStream_t s, NormArgs& a, const Rotation& rot, int* blocks) {
  for (int w = 0; w < 2; ++w) {
    a.vary_tokens[w][0] = along_tokens(a.x[w]);
    a.vary_tokens[w][1] = along_tokens(a.g[w]);
    a.vary_tokens[w][2] = along_tokens(a.y[w]);
  }
  const int pitch = a.P | 1;
  const size_t smem = sizeof(float) * ((((BWD ? 2 : 1) * kTokens * pitch + 1) & ~1) + kTokens * a.rotary);
  SB_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(norm_tile_kernel<BWD>), 100 * 1024));
  *blocks = std::min((a.tokens + kTokens - 1) / kTokens, kMaxPartials);
  SB_LAUNCH_OK(launch_k(norm_tile_kernel<BWD>, *blocks, 256, smem, s, a, turns_of(rot)));
  return SB_OK;
}

}  // namespace

size_t qk_norm_scratch_bytes() { return sizeof(float) * 2 * kNormMaxHead * kMaxPartials; }

int launch_qk_norm_fwd(cudaStream_t s, Proj q, Proj k, const void* q_gain, const void* k_gain, View2 pos, Proj q_out, Proj k_out,
                       const Rotation& rot) {
  NormArgs a = norm_args(q, k, q_gain, k_gain, pos, rot);
  if (a.tokens == 0) return SB_OK;
  a.y[0] = q_out; a.y[1] = k_out;
  int blocks;
  return launch_tiles<false>(s, a, rot, &blocks);
}

int launch_qk_norm_bwd(cudaStream_t s, void* scratch, Proj dq_out, Proj dk_out, Proj q, Proj k, const void* q_gain, const void* k_gain,
                       View2 pos, Proj dq, Proj dk, void* dq_gain, void* dk_gain, const Rotation& rot) {
  NormArgs a = norm_args(q, k, q_gain, k_gain, pos, rot);
  a.g[0] = dq_out; a.g[1] = dk_out;
  a.y[0] = dq; a.y[1] = dk;
  a.partial = reinterpret_cast<float*>(scratch);
  int blocks = 0;                        // without tokens the gains' gradients are 0
  if (a.tokens > 0) SB_TRY(launch_tiles<true>(s, a, rot, &blocks));
  SB_LAUNCH_OK(launch_k(gain_finish_kernel, dim3((a.P + 31) / 32, k.H > 0 ? 2 : 1), 512, 0, s, a.partial, blocks, a.P,
                        reinterpret_cast<sb_half*>(dq_gain), reinterpret_cast<sb_half*>(dk_gain)));
  return SB_OK;
}

}  // namespace sb
