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
  Proj q, k, v, o, g;
  RelRows lse;
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
__device__ __forceinline__ int first_of(const AttnArgs& a, int b) {
  return a.first ? max(-(1 << 29), min(1 << 29, a.first[b])) : 0;
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

// What the backward pass knows of 64 query rows (RelBackward in ops.h); four threads a row.  `vec`: both tensors have unit-stride
// features in 16-byte pieces; else lanes run along rows.
__global__ void __launch_bounds__(256)
row_records_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, float* records, int* next, int vec) {
  __shared__ float part[4][64];
  grid_dependency_sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) *next = 0;
  const int blocks = (a.J + 63) / 64;
  const long long all = (long long)a.H * a.B * blocks;
  for (long long it = blockIdx.x; it < all; it += gridDim.x) {
    const int j0 = (int)(it % blocks) * 64, h = (int)(it / blocks % a.H), b = (int)(it / blocks / a.H);
    const int row = vec ? threadIdx.x >> 2 : threadIdx.x & 63, i = vec ? threadIdx.x & 3 : threadIdx.x >> 6;
    float sum = 0.f;
    if (j0 + row < a.J) {
      const sb_half* g = row_of(a.g, h, b, j0 + row);
      const sb_half* o = row_of(a.o, h, b, j0 + row);
      if (vec) {
        for (int p = i * 8; p < a.P; p += 32) {
          float x[8], y[8];
          unpack8(*reinterpret_cast<const uint4*>(g + p), x);
          unpack8(*reinterpret_cast<const uint4*>(o + p), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x[e], y[e], sum);
        }
      } else {
        for (int p = i; p < a.P; p += 4) sum = fmaf(sb_h2f(g[p * a.g.sP]), sb_h2f(o[p * a.o.sP]), sum);
      }
    }
    __syncthreads();
    part[i][row] = sum;
    __syncthreads();
    if (threadIdx.x < 64) {
      const int j = j0 + threadIdx.x;
      float lse = INFINITY, weight = 0.f;
      if (j < a.J) {
        lse = a.lse.p[h * a.lse.sH + b * a.lse.sB + j * a.lse.sJ] * 1.4426950408889634f;
        if (lse == -INFINITY) lse = INFINITY;
        const int pos = first_of(a, b) + j;
        int n = keys_of(a, b);
        if (a.causal) n = max(0, min(n, pos + 1));
        // a row's score gradients sum to zero, so a row whose keys all share a bucket adds nothing to the table: its sum would
        // only be what D, from the rounded output, is off by
        if (n > 0 && bucket_of(a, st, -pos) != bucket_of(a, st, n - 1 - pos)) weight = 1.f;
      }
      float* r = records + it * 192 + threadIdx.x;
      r[0] = lse;
      r[64] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
      r[128] = weight;
    }
  }
}

// dtable[n,h] = the head's sums over the relative positions of bucket n; one block each, in a fixed order.
__global__ void __launch_bounds__(128)
table_finish_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, const float* partial, int rows, int reach,
                    sb_half* out, long long sN, long long sH) {
  __shared__ float part[4];
  grid_dependency_sync();
  const int n = blockIdx.x, h = blockIdx.y, entries = 2 * reach + 1;
  const bool behind = n >= a.n;
  const int i = behind ? n - a.n : n;
  // distances [lo, hi]; without `bidirectional` every key behind the query has distance 0
  int lo = st.s[i], hi = i + 1 < a.n ? st.s[i + 1] - 1 : reach;
  if (behind) lo = max(lo, 1);
  hi = min(hi, reach);
  int from = behind ? reach + lo : reach - hi, to = behind ? reach + hi : reach - lo;
  if (!a.bidirectional && lo == 0 && hi >= 0) to = 2 * reach;
  const int run = max(0, to - from + 1);
  const float* base = partial + (long long)h * rows * entries + from;
  const long long all = (long long)rows * run;
  float s = 0.f;
#pragma unroll 4
  for (long long e = threadIdx.x; e < all; e += 128) s += base[e / run * entries + e % run];
  s = group_sum<32>(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) out[n * sN + h * sH] = sb_f2h((part[0] + part[1]) + (part[2] + part[3]));
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

namespace {
// and for the backward pass records, sums and the queue's counter
struct BwdPlan { Plan p; size_t records, partial, next, bytes; int rows; };
BwdPlan bwd_plan(const Proj& dout, const Proj& q, const Proj& k, const Proj& v, const RelBias& bias) {
  BwdPlan b;
  b.p = plan_of({&dout, &q, &k, &v}, q.H, bias);
  b.rows = q.B * ((q.R + 127) / 128) * 2;
  b.records = b.p.bytes;
  b.partial = b.records + align256(sizeof(float) * 192 * (size_t)q.H * q.B * ((q.R + 63) / 64));
  b.next = b.partial + align256(sizeof(float) * (size_t)q.H * b.rows * (2 * b.p.reach + 1));
  b.bytes = b.next + 256;
  return b;
}
}  // namespace

size_t rel_attn_bwd_scratch_bytes(const Proj& dout, const Proj& q, const Proj& k, const Proj& v, const RelBias& bias) {
  return bwd_plan(dout, q, k, v, bias).bytes;
}

int launch_rel_attn_bwd(cudaStream_t s, void* scratch, Proj dout, Proj q, Proj k, Proj v, const RelBias& bias, Proj out, RelRows lse,
                        Proj dq, Proj dk, Proj dv, void* dtable, long long dt_sN, long long dt_sH, const RelSpan& span) {
  Starts st;
  AttnArgs a = attn_args(q, k, v, bias, out, lse, span, &st);
  a.g = dout;
  const BwdPlan pl = bwd_plan(dout, q, k, v, bias);
  char* base = reinterpret_cast<char*>(scratch);
  RelTables t;
  SB_TRY(expand_bias(s, a, st, scratch, pl.p, &t));
  auto pieces = [](const Proj& x) {
    return x.sP == 1 && x.P % 8 == 0 && !((x.sH | x.sB | x.sR) & 7) && !(reinterpret_cast<uintptr_t>(x.p) & 15u);
  };
  float* records = reinterpret_cast<float*>(base + pl.records);
  int* next = reinterpret_cast<int*>(base + pl.next);
  const long long blocks = (long long)a.H * a.B * ((a.J + 63) / 64);
  SB_LAUNCH_OK(launch_k(row_records_kernel, (unsigned)std::min<long long>(blocks, 8 * usable_sms(device_facts().sms)), 256, 0, s, a, st, records,
                        next, pieces(dout) && pieces(out) ? 1 : 0));
  SB_TRY(direct_or_packed(s, scratch, pl.p.at[0], &dout));
  SB_TRY(direct_or_packed(s, scratch, pl.p.at[1], &q));
  SB_TRY(direct_or_packed(s, scratch, pl.p.at[2], &k));
  SB_TRY(direct_or_packed(s, scratch, pl.p.at[3], &v));
  float* partial = reinterpret_cast<float*>(base + pl.partial);
  SB_TRY(launch_rel_tiles_bwd(s, dout, q, k, v, t, RelBackward{records, partial, next}, dq, dk, dv, span));
  SB_LAUNCH_OK(launch_k(table_finish_kernel, dim3(a.buckets, a.H), 128, 0, s, a, st, partial, pl.rows, pl.p.reach,
                        reinterpret_cast<sb_half*>(dtable), dt_sN, dt_sH));
  return SB_OK;
}

}  // namespace sb
