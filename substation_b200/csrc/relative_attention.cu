// Attention with a learned bias per head and bucket of relative positions (sb_relative_attention; formulas in the header).

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "ops.h"

namespace sb {

namespace {

constexpr int kMaxP = kRelMaxHead;
constexpr int kRelPad = 160;                        // as the tile kernels' kPad
constexpr float kHidden = -8.507059173023462e37f;   // -2^126: entries at or below hide their keys

struct Starts { int s[kRelMaxBuckets]; };
struct AttnArgs {
  Proj q, k, v, o, g, dq, dk, dv;
  RelRows lse;
  float* dsum;              // [H][B][J]
  float* partial;           // [H][B][row blocks][buckets]
  const sb_half* table;
  long long t_sN, t_sH;
  int n, bidirectional, buckets;
  float scale;
  int causal;
  const int* lengths;
  const int* first;
  int J, K, H, G, B, P;
};

__device__ __forceinline__ int bucket_of(const AttnArgs& a, const Starts& st, int rel) {
  const int d = rel > 0 ? (a.bidirectional ? rel : 0) : -rel;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (st.s[mid] <= d) lo = mid; else hi = mid - 1;
  }
  return lo + (a.bidirectional && rel > 0 ? a.n : 0);
}
__device__ __forceinline__ const sb_half* row_of(const Proj& v, int h, int b, int r) {
  return reinterpret_cast<const sb_half*>(v.p) + (long long)h * v.sH + (long long)b * v.sB + (long long)r * v.sR;
}
__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  return a.lengths ? max(0, min(a.K, a.lengths[b])) : a.K;
}

// rows[h][i] = log2(e) * bias of head h at relative position i - kRelPad - reach, which stays at its end values beyond the reach.
// Finite biases stay finite, so that a row of nothing but the lowest ones still has a maximum.
__global__ void __launch_bounds__(256)
expand_bias_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, float* rows, int pitch, int reach) {
  grid_dependency_sync();
  const int i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (i >= pitch) return;
  const int rel = max(-reach, min(reach, i - kRelPad - reach));
  const float b = sb_h2f(a.table[bucket_of(a, st, rel) * a.t_sN + h * a.t_sH]);
  rows[(long long)h * pitch + i] = b <= kHidden ? -INFINITY : b * 1.4426950408889634f;
}

// [P,H,B,R] of any strides -> [B][H][R][Pp], which tensor maps can address; 64 rows of one head and sample a block.
__global__ void __launch_bounds__(256)
pack_rows_kernel(const Proj x, sb_half* dst, int Pp, int along_rows) {
  __shared__ sb_half tile[64][kMaxP + 2];
  grid_dependency_sync();
  const int blocks = (x.R + 63) / 64;
  const long long all = (long long)x.H * x.B * blocks;
  for (long long it = blockIdx.x; it < all; it += gridDim.x) {
    const int r0 = (int)(it % blocks) * 64, h = (int)(it / blocks % x.H), b = (int)(it / blocks / x.H), n = min(64, x.R - r0);
    const sb_half* src = row_of(x, h, b, r0);
    __syncthreads();
    if (along_rows) {
      const int r = threadIdx.x & 63;
      if (r < n)
        for (int p = threadIdx.x >> 6; p < x.P; p += 4) tile[r][p] = src[p * x.sP + r * x.sR];
    } else {
      for (int r = threadIdx.x >> 5; r < n; r += 8)
        for (int p = threadIdx.x & 31; p < x.P; p += 32) tile[r][p] = src[p * x.sP + r * x.sR];
    }
    __syncthreads();
    sb_half* d = dst + (((long long)b * x.H + h) * x.R + r0) * Pp;
    for (int r = threadIdx.x >> 5; r < n; r += 8)
      for (int p = threadIdx.x & 31; p < x.P; p += 32) d[(long long)r * Pp + p] = tile[r][p];
  }
}

// dq, D and the table's sums: eight query rows of one head and sample per block, one warp each.
__global__ void __launch_bounds__(256)
simple_dq_kernel(const AttnArgs a, const Starts st) {
  extern __shared__ float smem[];
  float* bins = smem;                                  // [8][buckets]
  float* qs = bins + 8 * a.buckets;                    // [8][P]
  float* gs = qs + 8 * kMaxP;                          // [8][P]
  grid_dependency_sync();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks = (a.J + 7) / 8;
  const long long all = (long long)a.H * a.B * blocks;
  for (long long it = blockIdx.x; it < all; it += gridDim.x) {
    const int j = (int)(it % blocks) * 8 + w, b = (int)(it / blocks % a.B), h = (int)(it / blocks / a.B), hk = h / (a.H / a.G);
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * a.buckets; i += 256) bins[i] = 0.f;
    float dsum = 0.f;
    if (j < a.J)
      for (int p = lane; p < a.P; p += 32) {
        qs[w * kMaxP + p] = sb_h2f(row_of(a.q, h, b, j)[p * a.q.sP]);
        const float g = sb_h2f(row_of(a.g, h, b, j)[p * a.g.sP]);
        gs[w * kMaxP + p] = g;
        dsum = fmaf(g, sb_h2f(row_of(a.o, h, b, j)[p * a.o.sP]), dsum);
      }
    __syncthreads();
    dsum = group_sum<32>(dsum);
    if (j < a.J) {
      if (lane == 0) a.dsum[((long long)h * a.B + b) * a.J + j] = dsum;
      const float lse = a.lse.p[h * a.lse.sH + b * a.lse.sB + j * a.lse.sJ];
      const int pos = (a.first ? a.first[b] : 0) + j;
      int n = keys_of(a, b);
      if (a.causal) n = max(0, min(n, pos + 1));
      if (lse == -INFINITY) n = 0;
      // a row's ds sum to zero, so a row whose keys all share a bucket adds nothing to the table; its sum would be D's rounding
      const bool mixed = n > 0 && bucket_of(a, st, -pos) != bucket_of(a, st, n - 1 - pos);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k0 = 0; k0 < n; k0 += 32) {
        const int k = k0 + lane;
        float ds = 0.f;
        int bucket = 0;
        if (k < n) {
          const sb_half* kr = row_of(a.k, hk, b, k);
          const sb_half* vr = row_of(a.v, hk, b, k);
          float dot = 0.f, dp = 0.f;
          for (int p = 0; p < a.P; ++p) {
            dot = fmaf(qs[w * kMaxP + p], sb_h2f(kr[p * a.k.sP]), dot);
            dp = fmaf(gs[w * kMaxP + p], sb_h2f(vr[p * a.v.sP]), dp);
          }
          bucket = bucket_of(a, st, k - pos);
          const float bias = sb_h2f(a.table[bucket * a.t_sN + h * a.t_sH]);
          ds = bias <= kHidden ? 0.f : expf(fmaf(dot, a.scale, bias) - lse) * (dp - dsum);
        }
        for (int i = 0; i < min(32, n - k0); ++i) {
          const float d = __shfl_sync(0xffffffffu, ds, i);
          const int bk = __shfl_sync(0xffffffffu, bucket, i);
          const sb_half* kr = row_of(a.k, hk, b, k0 + i);
          if (lane == 0 && mixed) bins[w * a.buckets + bk] += d;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c * 32 + lane < a.P) acc[c] = fmaf(d, sb_h2f(kr[(c * 32 + lane) * a.k.sP]), acc[c]);
        }
      }
      sb_half* out = const_cast<sb_half*>(row_of(a.dq, h, b, j));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c * 32 + lane < a.P) out[(c * 32 + lane) * a.dq.sP] = sb_f2h(acc[c] * a.scale);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.buckets; i += 256) {
      float s = 0.f;
      for (int x = 0; x < 8; ++x) s += bins[x * a.buckets + i];
      a.partial[it * a.buckets + i] = s;
    }
  }
}

// One warp per key row: lanes along queries, then along features.
__global__ void __launch_bounds__(256)
simple_dkv_kernel(const AttnArgs a, const Starts st) {
  __shared__ float ks[8][kMaxP], vs[8][kMaxP];
  grid_dependency_sync();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.H / a.G;
  const long long rows = (long long)a.G * a.B * a.K;
  for (long long r = (long long)blockIdx.x * 8 + w; r < rows; r += (long long)gridDim.x * 8) {
    const int k = (int)(r % a.K), b = (int)(r / a.K % a.B), hk = (int)(r / a.K / a.B);
    float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
    if (k < keys_of(a, b)) {
      __syncwarp();
      for (int p = lane; p < a.P; p += 32) {
        ks[w][p] = sb_h2f(row_of(a.k, hk, b, k)[p * a.k.sP]);
        vs[w][p] = sb_h2f(row_of(a.v, hk, b, k)[p * a.v.sP]);
      }
      __syncwarp();
      const int first = a.first ? a.first[b] : 0;
      for (int h = hk * group; h < (hk + 1) * group; ++h)
        for (int j0 = 0; j0 < a.J; j0 += 32) {
          const int j = j0 + lane;
          float pr = 0.f, ds = 0.f;
          if (j < a.J && !(a.causal && k > first + j)) {
            const sb_half* qr = row_of(a.q, h, b, j);
            const sb_half* gr = row_of(a.g, h, b, j);
            float dot = 0.f, dp = 0.f;
            for (int p = 0; p < a.P; ++p) {
              dot = fmaf(ks[w][p], sb_h2f(qr[p * a.q.sP]), dot);
              dp = fmaf(vs[w][p], sb_h2f(gr[p * a.g.sP]), dp);
            }
            const float bias = sb_h2f(a.table[bucket_of(a, st, k - first - j) * a.t_sN + h * a.t_sH]);
            const float lse = a.lse.p[h * a.lse.sH + b * a.lse.sB + j * a.lse.sJ];
            pr = bias <= kHidden || lse == -INFINITY ? 0.f : expf(fmaf(dot, a.scale, bias) - lse);
            ds = pr * (dp - a.dsum[((long long)h * a.B + b) * a.J + j]);
          }
          for (int i = 0; i < min(32, a.J - j0); ++i) {
            const float x = __shfl_sync(0xffffffffu, pr, i), d = __shfl_sync(0xffffffffu, ds, i);
            const sb_half* qr = row_of(a.q, h, b, j0 + i);
            const sb_half* gr = row_of(a.g, h, b, j0 + i);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c * 32 + lane < a.P) {
                dv[c] = fmaf(x, sb_h2f(gr[(c * 32 + lane) * a.g.sP]), dv[c]);
                dk[c] = fmaf(d, sb_h2f(qr[(c * 32 + lane) * a.q.sP]), dk[c]);
              }
          }
        }
    }
    sb_half* ok = const_cast<sb_half*>(row_of(a.dk, hk, b, k));
    sb_half* ov = const_cast<sb_half*>(row_of(a.dv, hk, b, k));
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 32 + lane < a.P) {
        ok[(c * 32 + lane) * a.dk.sP] = sb_f2h(dk[c] * a.scale);
        ov[(c * 32 + lane) * a.dv.sP] = sb_f2h(dv[c]);
      }
  }
}

// dtable[n,h] = sum of the head's partial rows, one warp each in a fixed order.
__global__ void __launch_bounds__(256)
table_finish_kernel(const float* partial, int rows, int buckets, int H, sb_half* out, long long sN, long long sH) {
  grid_dependency_sync();
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= buckets * H) return;
  const int h = i / buckets, n = i % buckets;
  float s = 0.f;
  for (int r = lane; r < rows; r += 32) s += partial[((long long)h * rows + r) * buckets + n];
  s = group_sum<32>(s);
  if (lane == 0) out[n * sN + h * sH] = sb_f2h(s);
}

AttnArgs attn_args(const Proj& q, const Proj& k, const Proj& v, const RelBias& bias, const Proj& out, const RelRows& lse, const RelSpan& span,
                   Starts* st) {
  AttnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q; a.k = k; a.v = v; a.o = out; a.lse = lse;
  a.table = reinterpret_cast<const sb_half*>(bias.table);
  a.t_sN = bias.sN; a.t_sH = bias.sH;
  a.n = bias.n; a.bidirectional = bias.bidirectional; a.buckets = bias.bidirectional ? 2 * bias.n : bias.n;
  a.scale = span.scale; a.causal = span.causal; a.lengths = span.lengths; a.first = span.first;
  a.J = q.R; a.K = k.R; a.H = q.H; a.G = k.H; a.B = q.B; a.P = q.P;
  memset(st, 0, sizeof(*st));
  for (int i = 0; i < bias.n; ++i) st->s[i] = bias.starts[i];
  return a;
}
size_t dsum_bytes(const Proj& q) { return (sizeof(float) * (size_t)q.H * q.B * q.R + 255) / 256 * 256; }

// Scratch: rows of biases, then a packed copy of each operand that tensor maps cannot address.
struct Plan { int pitch, reach; size_t at[4], bytes; };
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
size_t packed_bytes(const Proj& x) { return align256(2 * (size_t)((x.P + 7) / 8 * 8) * x.H * x.B * x.R); }
Plan plan_of(std::initializer_list<const Proj*> operands, int heads, const RelBias& bias) {
  Plan p;
  p.reach = std::max(1, bias.starts[bias.n - 1]);
  p.pitch = (2 * p.reach + 1 + 2 * kRelPad + 3) / 4 * 4;
  p.bytes = align256(sizeof(float) * (size_t)p.pitch * heads);
  int i = 0;
  for (const Proj* x : operands) {
    p.at[i++] = p.bytes;
    if (!rel_direct(*x)) p.bytes += packed_bytes(*x);
  }
  return p;
}
// x as tensor maps can address it: itself, or the copy at `at`.
int direct_or_packed(cudaStream_t s, void* scratch, size_t at, Proj* x) {
  if (rel_direct(*x)) return SB_OK;
  const int Pp = (x->P + 7) / 8 * 8;
  auto mag = [](long long v) { return v < 0 ? -v : v; };
  sb_half* dst = reinterpret_cast<sb_half*>(reinterpret_cast<char*>(scratch) + at);
  const long long blocks = (long long)x->H * x->B * ((x->R + 63) / 64);
  SB_LAUNCH_OK(launch_k(pack_rows_kernel, (unsigned)std::min<long long>(blocks, 8 * usable_sms(device_facts().sms)), 256, 0, s, *x, dst, Pp,
                        x->R > 1 && mag(x->sR) < mag(x->sP) ? 1 : 0));
  x->p = dst;
  x->sP = 1; x->sR = Pp; x->sH = (long long)Pp * x->R; x->sB = x->sH * x->H;
  return SB_OK;
}
int expand_bias(cudaStream_t s, const AttnArgs& a, const Starts& st, void* scratch, const Plan& pl, RelTables* t) {
  t->rows = reinterpret_cast<float*>(scratch); t->pitch = pl.pitch; t->reach = pl.reach;
  SB_LAUNCH_OK(launch_k(expand_bias_kernel, dim3((pl.pitch + 255) / 256, a.H), 256, 0, s, a, st, reinterpret_cast<float*>(scratch), pl.pitch, pl.reach));
  return SB_OK;
}

}  // namespace

size_t rel_attn_scratch_bytes(const Proj& q, const Proj& k, const Proj& v, const RelBias& bias) { return plan_of({&q, &k, &v}, q.H, bias).bytes; }

int launch_rel_attn_fwd(cudaStream_t s, void* scratch, Proj q, Proj k, Proj v, const RelBias& bias, Proj out, RelRows lse, const RelSpan& span) {
  Starts st;
  const AttnArgs a = attn_args(q, k, v, bias, out, lse, span, &st);
  const Plan pl = plan_of({&q, &k, &v}, q.H, bias);
  RelTables t;
  SB_TRY(expand_bias(s, a, st, scratch, pl, &t));
  SB_TRY(direct_or_packed(s, scratch, pl.at[0], &q));
  SB_TRY(direct_or_packed(s, scratch, pl.at[1], &k));
  SB_TRY(direct_or_packed(s, scratch, pl.at[2], &v));
  return launch_rel_tiles_fwd(s, q, k, v, t, out, lse, span);
}

size_t rel_attn_bwd_scratch_bytes(const Proj&, const Proj& q, const Proj&, const Proj&, const RelBias& bias) {
  return dsum_bytes(q) + sizeof(float) * (size_t)q.H * q.B * ((q.R + 7) / 8) * (bias.bidirectional ? 2 : 1) * bias.n;
}

int launch_rel_attn_bwd(cudaStream_t s, void* scratch, Proj dout, Proj q, Proj k, Proj v, const RelBias& bias, Proj out, RelRows lse,
                        Proj dq, Proj dk, Proj dv, void* dtable, long long dt_sN, long long dt_sH, const RelSpan& span) {
  Starts st;
  AttnArgs a = attn_args(q, k, v, bias, out, lse, span, &st);
  a.g = dout; a.dq = dq; a.dk = dk; a.dv = dv;
  a.dsum = reinterpret_cast<float*>(scratch);
  a.partial = reinterpret_cast<float*>(reinterpret_cast<char*>(scratch) + dsum_bytes(q));
  const int blocks = (a.J + 7) / 8;
  const size_t smem = sizeof(float) * (8 * a.buckets + 16 * kMaxP);
  SB_LAUNCH_OK(launch_k(simple_dq_kernel, (unsigned)std::min<long long>((long long)a.H * a.B * blocks, 1184), 256, smem, s, a, st));
  SB_LAUNCH_OK(launch_k(simple_dkv_kernel, (unsigned)std::min<long long>(((long long)a.G * a.B * a.K + 7) / 8, 1184), 256, 0, s, a, st));
  SB_LAUNCH_OK(launch_k(table_finish_kernel, (unsigned)((a.buckets * a.H + 7) / 8), 256, 0, s, a.partial, a.B * blocks, a.buckets, a.H,
                        reinterpret_cast<sb_half*>(dtable), dt_sN, dt_sH));
  return SB_OK;
}

}  // namespace sb
