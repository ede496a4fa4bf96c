// Attention with a learned bias per head and bucket of relative positions (sb_relative_attention; formulas in the header).

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "ops.h"

namespace sb {

namespace {

constexpr int kMaxP = kRelMaxHead;
constexpr int kRelPad = 96;                         // as the tile kernels' kPad
constexpr float kHidden = -8.507059173023462e37f;   // -2^126: entries at or below hide their keys
constexpr float kLargest = 1.7014118346046923e38f;   // 2^127: entries above count as this, so that log2(e) of them is finite and leaves room

// A table's entry in units of log2.
__device__ __forceinline__ float bias_of_entry(sb_half entry) {
  const float b = sb_h2f(entry);
  return b <= kHidden ? -INFINITY : (b > kLargest ? kLargest : b) * 1.4426950408889634f;
}

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

__device__ __forceinline__ int bucket_of(const AttnArgs& a, const int* starts, int rel) {
  const int d = rel > 0 ? (a.bidirectional ? rel : 0) : -rel;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= d) lo = mid; else hi = mid - 1;
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
// Biases stay finite, so that a row of nothing but float16's lowest still has a maximum.
// Block `part` of expand_blocks() for the head.  A launch and a search among the starts: 1.9 us alone, whatever the size.
struct Expand { float* rows; int pitch, reach; int* next; };   // next: the work queue of the kernel that follows
__host__ __device__ constexpr int expand_blocks(int pitch) { return (pitch + 255) / 256; }
__device__ __forceinline__ void expand_part(const AttnArgs& a, const int* starts, const Expand& x, int h, int part) {
  if (h == 0 && part == 0 && threadIdx.x == 0) *x.next = 0;
  const int i = part * 256 + threadIdx.x;
  if (i >= x.pitch) return;
  const int rel = max(-x.reach, min(x.reach, i - kRelPad - x.reach));
  x.rows[(long long)h * x.pitch + i] = bias_of_entry(a.table[bucket_of(a, starts, rel) * a.t_sN + h * a.t_sH]);
}
__global__ void __launch_bounds__(256)
expand_bias_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, const __grid_constant__ Expand x) {
  grid_dependency_sync();
  expand_part(a, st.s, x, blockIdx.y, blockIdx.x);
}

// Copies of operands that tensor maps cannot address: [P,H,B,R] of any strides -> [B][H][R][Pp], up to four of them in a launch.  A
// block turns 64 rows of one head and sample over in shared memory: words of two rows where rows lie side by side in them, else
// elements along rows or along features, 16 of them on their way per thread, and 16-byte pieces out.  B=8, L=512, three operands of
// 16 heads of 64 (50 MB): 13 us head-first, 15 feature-innermost off the 16-byte grid (26 and 40 with one load after the other and a
// launch each); bound by the rounds of loads that its blocks wait for.
enum { kPackTwos, kPackRows, kPackFeatures };
struct PackJobs {
  struct { Proj x; sb_half* dst; int mode; int first; } job[4];   // first: its first block
  int n, blocks;
};
__global__ void __launch_bounds__(256, 5)
pack_rows_kernel(const __grid_constant__ PackJobs jobs) {
  constexpr int kPitch = kMaxP + 8;                            // (pieces aligned, rows four banks apart)
  __shared__ __align__(16) sb_half tile[64][kPitch];
  grid_dependency_sync();
  int n = 0;
  while (n + 1 < jobs.n && (int)blockIdx.x >= jobs.job[n + 1].first) ++n;
  const Proj& x = jobs.job[n].x;
  const int blocks = (x.R + 63) / 64, it = blockIdx.x - jobs.job[n].first, mode = jobs.job[n].mode;
  const int r0 = it % blocks * 64, h = it / blocks % x.H, b = it / blocks / x.H, rows = min(64, x.R - r0), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int Pp = (x.P + 7) / 8 * 8;
  const sb_half* src = row_of(x, h, b, r0);
  if (mode == kPackTwos) {                                    // a warp: 16 rows of four features
    const int r = (warp & 3) * 16 + (lane & 7) * 2, f = (warp >> 2) * 4 + (lane >> 3);
    const sb_half* at = src + f * x.sP + r;
    if (r < rows)
      for (int p0 = f; p0 < x.P; p0 += 64) {
        sb_half2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k, at += 8 * x.sP)
          if (p0 + k * 8 < x.P) v[k] = *reinterpret_cast<const sb_half2*>(at);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const sb_half* e = reinterpret_cast<const sb_half*>(&v[k]);
          if (p0 + k * 8 < x.P) tile[r][p0 + k * 8] = e[0];
          if (p0 + k * 8 < x.P) tile[r + 1][p0 + k * 8] = e[1];
        }
      }
  } else if (mode == kPackRows) {                             // a warp: 16 rows of two features
    const int r = (warp & 3) * 16 + (lane & 15), f = (warp >> 2) * 2 + (lane >> 4);
    const sb_half* at = src + f * x.sP + r * x.sR;
    if (r < rows)
      for (int p0 = f; p0 < x.P; p0 += 64) {
        sb_half v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k, at += 4 * x.sP)
          if (p0 + k * 4 < x.P) v[k] = *at;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (p0 + k * 4 < x.P) tile[r][p0 + k * 4] = v[k];
      }
  } else {                                                    // a warp: 32 features of a row
    const int f = (warp & 1) * 32 + lane, w = warp >> 1;
    for (int p = f; p < x.P; p += 64) {
      const sb_half* at = src + p * x.sP + w * x.sR;
      sb_half v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k, at += 4 * x.sR)
        if (w + k * 4 < rows) v[k] = *at;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (w + k * 4 < rows) tile[w + k * 4][p] = v[k];
    }
  }
  __syncthreads();
  sb_half* d = jobs.job[n].dst + (((long long)b * x.H + h) * x.R + r0) * Pp;
  const int pieces = Pp / 8;
  for (int i = threadIdx.x; i < rows * pieces; i += 256)
    *reinterpret_cast<uint4*>(d + i * 8) = *reinterpret_cast<const uint4*>(&tile[i / pieces][i % pieces * 8]);
}

// ---- few queries ------------------------------------------------------------------------------------------------
// The rows of a key head are the queries of all heads that share it, J for each.  A CTA takes 16 of them (one mma.sync tile) and a
// share of the keys; its four warps walk pieces of those keys in turn, each with a ring of its own filled by cp.async (which
// also puts zeros behind a sequence's end), softmax state and accumulator, joined at the end.  With more than one share, a
// second kernel joins those.  Bound by reading keys and values once (B=16, 32 heads on 8, 8192 keys of 128 features: 72 us, 87 % of the
// copy bandwidth); tcgen05's smallest tile would be 64 or 128 rows for the one to 16 there are, and the matrix work here
// is a few percent of the time.
constexpr int kFewThreads = 128;
constexpr float kFewRaise = kRelScaled ? 15.f : 0.f;   // exponentials, at most one here, are times 2^kFewRaise (see kRaise of the tile kernels)
template <int P>
struct FewCfg {
  static constexpr int kKeys = P == 64 ? 32 : 16;    // of a piece
  static constexpr int kStages = 3;
  static constexpr int kHalf = kKeys * P * 2;        // bytes of a piece's keys
  // A ring has a slot for each of its warp's pieces, up to kStages: short shares leave room for more CTAs.
  static constexpr int slots(int share) { return share <= 4 * kKeys ? 1 : share <= 8 * kKeys ? 2 : kStages; }
  static constexpr int smem(int share) {
    const int rings = 4 * slots(share) * 2 * kHalf, results = 4 * (16 * P + 32) * 4;
    return rings > results ? rings : results;
  }
};
struct FewParams {
  AttnArgs a;
  int rows, blocks, splits, reach, slots;            // rows of a key head, blocks of 16 of them; slots of a ring
  int before, behind;                                // buckets of far keys
  float* partial;                                    // [B][G][rows][splits][P + 2]: output, reference, sum; null with one share
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
#ifdef SB_BF16
#define SB_MMA_TYPES "f32.bf16.bf16.f32"
#else
#define SB_MMA_TYPES "f32.f16.f16.f32"
#endif
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col." SB_MMA_TYPES " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_pair(float x, float y) {
  const sb_half2 h = sb_f2h2(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__host__ __device__ constexpr int share_of(int keys, int splits) { return ((keys + splits - 1) / splits + 31) & ~31; }
template <int P>
__global__ void __launch_bounds__(kFewThreads)
few_queries_kernel(const __grid_constant__ FewParams p, const __grid_constant__ Starts st) {
  using Cfg = FewCfg<P>;
  constexpr int kKeys = Cfg::kKeys, kStages = Cfg::kStages, kSteps = P / 16, kTiles = kKeys / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int starts[kRelMaxBuckets];
  __shared__ uint16_t map[2 * kRelMaxReach + 2];
  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_sync();
  const int split = blockIdx.x % p.splits, block = blockIdx.x / p.splits % p.blocks, unit = blockIdx.x / p.splits / p.blocks;
  const int hk = unit % a.G, b = unit / a.G, rep = a.H / a.G;
  const int first = first_of(a, b);
  // keys that some row of the sample sees, and this CTA's share of them
  int keys = keys_of(a, b);
  if (a.causal) keys = max(0, min(keys, first + a.J));
  const int share = share_of(keys, p.splits);
  const int k_from = min(keys, split * share), k_to = min(keys, k_from + share);
  const int pieces = (k_to - k_from + kKeys - 1) / kKeys, mine = pieces > warp ? (pieces - warp + 3) >> 2 : 0;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * p.slots * 2 * Cfg::kHalf;
  const sb_half* kp = row_of(a.k, hk, b, 0);
  const sb_half* vp = row_of(a.v, hk, b, 0);

  // piece i of this warp into its slot: 16-byte chunk c of row r at c ^ (r & 7); a lane has one c and every kStep-th row
  constexpr int kStep = 32 / (P / 8);
  const int fr = lane / (P / 8), fc = lane % (P / 8), bytes = max(0, min(16, (a.P - fc * 8) * 2));
  const sb_half* fk = kp + (long long)(k_from + warp * kKeys + fr) * a.k.sR + (bytes > 0 ? fc * 8 : 0);
  const sb_half* fv = vp + (long long)(k_from + warp * kKeys + fr) * a.v.sR + (bytes > 0 ? fc * 8 : 0);
  int left = k_to - (k_from + warp * kKeys) - fr, slot = 0;
  auto fetch = [&](int i) {
    if (i < mine) {
      const uint32_t at = ring + slot * 2 * Cfg::kHalf;
#pragma unroll
      for (int x = 0; x < kKeys / kStep; ++x) {
        const int r = fr + x * kStep;
        const bool there = x * kStep < left;                 // (a row that is not there is read as no bytes of the first one)
        const uint32_t d = at + r * (P * 2) + ((fc ^ (r & 7)) << 4);
        cp_async16(d, there ? fk + (long long)(x * kStep) * a.k.sR : kp, there ? bytes : 0);
        cp_async16(d + Cfg::kHalf, there ? fv + (long long)(x * kStep) * a.v.sR : vp, there ? bytes : 0);
      }
      fk += (long long)(4 * kKeys) * a.k.sR;
      fv += (long long)(4 * kKeys) * a.v.sR;
      left -= 4 * kKeys;
      if (++slot == kStages) slot = 0;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  for (int i = threadIdx.x; i < a.n; i += kFewThreads) starts[i] = st.s[i];

  // this lane's two rows: queries as operands, positions, biases outside the varying part
  const int r0 = block * 16 + (lane >> 2);
  uint32_t qf[kSteps][4];
  int pos[2], head[2];
  float lo[2], hi[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = r0 + 8 * x, rc = min(r, p.rows - 1), j = rc % a.J;
    head[x] = hk * rep + rc / a.J;
    pos[x] = first + j;
    const sb_half* q = row_of(a.q, head[x], b, j);
    const int f = (lane & 3) * 2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int e = s * 16 + y * 8 + f;
        float u = 0.f, v = 0.f;
        if (r < p.rows && e < a.P) u = sb_h2f(q[e * a.q.sP]);
        if (r < p.rows && e + 1 < a.P) v = sb_h2f(q[(e + 1) * a.q.sP]);
        qf[s][y * 2 + x] = pack_pair(u, v);
      }
  }
  auto bias_of = [&](int bucket, int h) { return bias_of_entry(a.table[bucket * a.t_sN + h * a.t_sH]); };
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    lo[x] = bias_of(p.before, head[x]);
    hi[x] = bias_of(p.behind, head[x]);
  }
  __syncthreads();
  // buckets of the relative positions within reach, where this CTA's pieces have any
  const int pos_lo = first, pos_hi = first + a.J - 1;
  if (k_from + pieces * kKeys - 1 - pos_lo > -p.reach && k_from - pos_hi < p.reach) {
    for (int i = threadIdx.x; i <= 2 * p.reach; i += kFewThreads) map[i] = (uint16_t)bucket_of(a, starts, i - p.reach);
    __syncthreads();
  }
  const float c2 = a.scale * 1.4426950408889634f;
  float o[P / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < P / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  for (int i = 0; i < mine; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    fetch(i + kStages - 1);
    const int k0 = k_from + (warp + 4 * i) * kKeys;
    const uint32_t ks = ring + (i % kStages) * 2 * Cfg::kHalf, vs = ks + Cfg::kHalf;
    float s[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
    for (int t = 0; t < kTiles; t += 2)
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        uint32_t f[4];
        const int r = t * 8 + (lane & 7) + ((lane >> 4) << 3), ch = c * 2 + ((lane >> 3) & 1);
        ldsm4(ks + r * (P * 2) + ((ch ^ (r & 7)) << 4), f);
        mma16816(s[t], qf[c], f[0], f[1]);
        mma16816(s[t + 1], qf[c], f[2], f[3]);
      }
    // biases, what is hidden, maxima.  (All loads of biases unconditional: a branch for each waits for each)
    const bool near = k0 + kKeys - 1 - pos_lo > -p.reach && k0 - pos_hi < p.reach;
    const bool after = k0 - pos_hi >= p.reach, whole = k0 + kKeys <= k_to && !(a.causal && k0 + kKeys - 1 > pos_lo);
    float mx[2] = {-INFINITY, -INFINITY};
    const float flat[2] = {after ? hi[0] : lo[0], after ? hi[1] : lo[1]};
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = fmaf(s[t][e], c2, near ? 0.f : flat[e >> 1]);
    if (near) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = e >> 1, rel = k0 + t * 8 + (lane & 3) * 2 + (e & 1) - pos[x];
          s[t][e] += bias_of(map[max(-p.reach, min(p.reach, rel)) + p.reach], head[x]);
        }
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = k0 + t * 8 + (lane & 3) * 2 + (e & 1);
          if (k >= k_to || (a.causal && k > pos[e >> 1])) s[t][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
    bool raise = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
      raise |= mx[x] > m[x];
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float now = fmaxf(m[x], mx[x]), f = now == -INFINITY ? 1.f : ex2_unit(m[x] - now);
        m[x] = now;
        l[x] *= f;
#pragma unroll
        for (int t = 0; t < P / 8; ++t) {
          o[t][2 * x] *= f;
          o[t][2 * x + 1] *= f;
        }
      }
    }
    const float ref[2] = {(m[0] == -INFINITY ? 0.f : m[0]) - kFewRaise, (m[1] == -INFINITY ? 0.f : m[1]) - kFewRaise};
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[t][e] = ex2_unit(s[t][e] - ref[e >> 1]);
        l[e >> 1] += s[t][e];
      }
#pragma unroll
    for (int c = 0; c < kKeys / 16; ++c) {
      const uint32_t pf[4] = {pack_pair(s[2 * c][0], s[2 * c][1]), pack_pair(s[2 * c][2], s[2 * c][3]),
                              pack_pair(s[2 * c + 1][0], s[2 * c + 1][1]), pack_pair(s[2 * c + 1][2], s[2 * c + 1][3])};
#pragma unroll
      for (int t = 0; t < P / 8; t += 2) {
        uint32_t f[4];
        const int r = c * 16 + (lane & 15), ch = t + (lane >> 4);
        ldsm4_t(vs + r * (P * 2) + ((ch ^ (r & 7)) << 4), f);
        mma16816(o[t], pf, f[0], f[1]);
        mma16816(o[t + 1], pf, f[2], f[3]);
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // the warps' results side by side: output [4][16][P], then references and sums [4][16]
  float* so = reinterpret_cast<float*>(smem);
  float* sm = so + 4 * 16 * P;
  float* sl = sm + 64;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    const int r = (lane >> 2) + 8 * x;
    if ((lane & 3) == 0) {
      sm[warp * 16 + r] = m[x];
      sl[warp * 16 + r] = l[x];
    }
#pragma unroll
    for (int t = 0; t < P / 8; ++t)
      *reinterpret_cast<float2*>(so + (warp * 16 + r) * P + t * 8 + (lane & 3) * 2) = make_float2(o[t][2 * x], o[t][2 * x + 1]);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * P; x += kFewThreads) {
    const int r = x / P, f = x % P, row = block * 16 + r;
    if (row >= p.rows) break;
    float mm = sm[r];
#pragma unroll
    for (int w = 1; w < 4; ++w) mm = fmaxf(mm, sm[w * 16 + r]);
    float sum = 0.f, v = 0.f;
    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = ex2_unit(sm[w * 16 + r] - ref);
      sum = fmaf(sl[w * 16 + r], e, sum);
      v = fmaf(so[(w * 16 + r) * P + f], e, v);
    }
    const int h = hk * rep + row / a.J, j = row % a.J;
    if (p.partial) {
      float* d = p.partial + (((long long)unit * p.rows + row) * p.splits + split) * (P + 2);
      d[f] = v;
      if (f == 0) {
        d[P] = mm;
        d[P + 1] = sum;
      }
    } else {
      if (f < a.P) const_cast<sb_half*>(row_of(a.o, h, b, j))[f * a.o.sP] = sb_f2h(sees_none(sum) ? 0.f : v / sum);
      if (f == 0 && a.lse.p) a.lse.p[h * a.lse.sH + b * a.lse.sB + j * a.lse.sJ] = sees_none(sum) ? -INFINITY : (mm + (log2f(sum) - kFewRaise)) * 0.6931471805599453f;
    }
  }
}

// One warp per row joins its shares: with weights exp(reference - highest reference), sums and outputs add up.  Latency: 4 us for 512 rows
// of 128 features in two shares.
template <int P>
__global__ void __launch_bounds__(128)
join_splits_kernel(const __grid_constant__ FewParams p) {
  grid_dependency_sync();
  const AttnArgs& a = p.a;
  const long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (it >= (long long)a.B * a.G * p.rows) return;
  const int row = (int)(it % p.rows), unit = (int)(it / p.rows), hk = unit % a.G, b = unit / a.G;
  const int h = hk * (a.H / a.G) + row / a.J, j = row % a.J;
  const float* src = p.partial + it * p.splits * (P + 2);
  float mm = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) mm = fmaxf(mm, src[s * (P + 2) + P]);
  mm = group_max<32>(mm);
  float sum = 0.f, v[P / 32];
  const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
  for (int c = 0; c < P / 32; ++c) v[c] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* d = src + s * (P + 2);
    const float e = ex2_unit(d[P] - ref);
    sum = fmaf(d[P + 1], e, sum);
#pragma unroll
    for (int c = 0; c < P / 32; ++c) v[c] = fmaf(d[c * 32 + lane], e, v[c]);
  }
  sb_half* out = const_cast<sb_half*>(row_of(a.o, h, b, j));
#pragma unroll
  for (int c = 0; c < P / 32; ++c)
    if (c * 32 + lane < a.P) out[(c * 32 + lane) * a.o.sP] = sb_f2h(sees_none(sum) ? 0.f : v[c] / sum);
  if (lane == 0 && a.lse.p) a.lse.p[h * a.lse.sH + b * a.lse.sB + j * a.lse.sJ] = sees_none(sum) ? -INFINITY : (mm + (log2f(sum) - kFewRaise)) * 0.6931471805599453f;
}

// What the backward pass knows of 64 query rows (RelBackward in ops.h), four threads a row, and in the blocks before those the rows
// of biases.  `vec`, `vec_v`: dout and out, and v, have unit-stride features in 16-byte pieces; else lanes run along rows.  Bound by
// reading dout and out once (B=96, L=128, 16 heads of 64, 50 MB: 11 us, 70 % of the copy bandwidth), so everything is asked for before
// anything is waited for: one trip to memory a block (18 us with a barrier before the sums and another trip behind it).  VALUES, float16
// only: block n also looks at the n-th 64 rows of v, so that they are under way beside the rest; there are as many blocks as the longer of
// the two needs.  Maxima go out per warp, without a barrier (2 us less at B=96).
__device__ __forceinline__ float sum_of_four(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float2 add_squares(const float (&v)[8], float2 sum) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 x = make_float2(v[e], v[e + 1]);
    sum = fma2(x, x, sum);
  }
  return sum;
}
// The largest of a warp's values, none negative, to the warp's place; what is not finite does not count.
__device__ __forceinline__ void store_largest(float value, float* to) {
  const uint32_t most = __reduce_max_sync(0xffffffffu, value < INFINITY ? __float_as_uint(value) : 0u);
  if ((threadIdx.x & 31) == 0) to[threadIdx.x >> 5] = __uint_as_float(most);
}
template <int P, bool VALUES>
__global__ void __launch_bounds__(256, VALUES ? (P == 64 ? 4 : 2) : 1)
row_records_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, const __grid_constant__ Expand x, float* records, float* sizes,
                   int vec, int vec_v, int expanding, int rows, int values) {
  __shared__ float part[3][4][64];
  grid_dependency_sync();
  const int it = (int)blockIdx.x - expanding;
  if (it < 0) {
    const int parts = expand_blocks(x.pitch);
    expand_part(a, st.s, x, blockIdx.x / parts, blockIdx.x % parts);
    return;
  }
  // blocks that run together share tokens, whose heads usually lie side by side
  const int blocks = (a.J + 63) / 64, blocks_v = (a.K + 63) / 64;
  const long long sizes_of_out = 8ll * a.B * a.H * blocks;
  const int vrow = vec_v ? threadIdx.x >> 2 : threadIdx.x & 63, vi = vec_v ? threadIdx.x & 3 : threadIdx.x >> 6;
  const int hk = it % a.G, bv = it / a.G / blocks_v, block_v = it / a.G % blocks_v, k = block_v * 64 + vrow;
  uint4 vv[P / 32];
  const sb_half* v = nullptr;                                // null behind the length
  if (VALUES && it < values && k < keys_of(a, bv)) v = row_of(a.v, hk, bv, k);
  if (VALUES && vec_v)
#pragma unroll
    for (int c = 0; c < P / 32; ++c) {
      const int p = vi * 8 + c * 32;
      vv[c] = make_uint4(0u, 0u, 0u, 0u);
      if (v && p < a.P) vv[c] = *reinterpret_cast<const uint4*>(v + p);
    }
  if (!VALUES || it < rows) {
    const int h = it % a.H, block = it / a.H % blocks, b = it / a.H / blocks;
    const int row = vec ? threadIdx.x >> 2 : threadIdx.x & 63, i = vec ? threadIdx.x & 3 : threadIdx.x >> 6, j = block * 64 + row;
    const bool live = j < a.J;
    const sb_half* g = row_of(a.g, h, b, live ? j : 0);
    const sb_half* o = row_of(a.o, h, b, live ? j : 0);
    uint4 gv[P / 32], ov[P / 32];
    if (vec)
#pragma unroll
      for (int c = 0; c < P / 32; ++c) {
        const int p = i * 8 + c * 32;
        gv[c] = ov[c] = make_uint4(0u, 0u, 0u, 0u);
        if (p < a.P) {
          gv[c] = *reinterpret_cast<const uint4*>(g + p);
          ov[c] = *reinterpret_cast<const uint4*>(o + p);
        }
      }
    float lse = 0.f;
    int n = 0, pos = 0;
    if (i == 0) {
      lse = a.lse.p[h * a.lse.sH + b * a.lse.sB + (live ? j : 0) * a.lse.sJ];
      n = keys_of(a, b);
      pos = first_of(a, b) + j;
    }
    float sum = 0.f, square_g = 0.f, square_o = 0.f;
    if (vec) {
      float2 of_g = make_float2(0.f, 0.f), of_o = of_g;
#pragma unroll
      for (int c = 0; c < P / 32; ++c) {
        float u[8], w[8];
        unpack8(gv[c], u);
        unpack8(ov[c], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(u[e], w[e], sum);
        if (kRelScaled) of_g = add_squares(u, of_g);
        if (VALUES) of_o = add_squares(w, of_o);
      }
      sum = sum_of_four(sum);
      if (kRelScaled) square_g = sum_of_four(of_g.x + of_g.y);
      if (VALUES) square_o = sum_of_four(of_o.x + of_o.y);
    } else {
#pragma unroll 4
      for (int p = i; p < a.P; p += 4) {
        const float u = sb_h2f(g[p * a.g.sP]), w = sb_h2f(o[p * a.o.sP]);
        sum = fmaf(u, w, sum);
        if (kRelScaled) square_g = fmaf(u, u, square_g);
        if (VALUES) square_o = fmaf(w, w, square_o);
      }
      part[0][i][row] = sum;
      if (kRelScaled) part[1][i][row] = square_g;
      if (VALUES) part[2][i][row] = square_o;
      __syncthreads();
      if (i == 0) {
        auto all = [&](const float (&l)[4][64]) { return (l[0][row] + l[1][row]) + (l[2][row] + l[3][row]); };
        sum = all(part[0]);
        if (kRelScaled) square_g = all(part[1]);
        if (VALUES) square_o = all(part[2]);
      }
    }
    if (i == 0) {
      if (a.causal) n = max(0, min(n, pos + 1));
      // a row's score gradients sum to zero, so a row whose keys all share a bucket adds nothing to the table: its sum would
      // only be what D, from the rounded output, is off by
      // (seldom; most rows have keys on both sides or, of the far ones, before and within the reach, and need no search)
      const int lo = -pos, hi = n - 1 - pos, last = st.s[a.n - 1];
      const bool sides = (a.bidirectional && lo <= 0 && hi > 0) || (last > 0 && lo <= -last && hi > -last);
      const bool alike = n <= 0 || (!sides && bucket_of(a, st.s, lo) == bucket_of(a, st.s, hi));
      float* r = records + (((long long)b * a.H + h) * blocks + block) * 192 + row;
      r[0] = live && lse != -INFINITY ? lse * 1.4426950408889634f : INFINITY;
      r[64] = live ? sum : 0.f;
      r[128] = live && alike ? 0.f : 1.f;
    }
    if (kRelScaled) {
      const bool counts = i == 0 && live && lse != -INFINITY;
      float* to = sizes + (((long long)b * a.H + h) * blocks + block) * 8;
      store_largest(counts ? square_g : 0.f, to);
      if (VALUES) store_largest(counts ? square_o : 0.f, to + sizes_of_out);
    }
  }
  if (VALUES && it < values) {
    float s = 0.f;
    if (vec_v) {
      float2 of_v = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < P / 32; ++c) {
        float u[8];
        unpack8(vv[c], u);
        of_v = add_squares(u, of_v);
      }
      s = sum_of_four(of_v.x + of_v.y);
    } else {
      if (v)
#pragma unroll 4
        for (int p = vi; p < a.P; p += 4) {
          const float u = sb_h2f(v[p * a.v.sP]);
          s = fmaf(u, u, s);
        }
      __syncthreads();                                       // (`part` may still be read)
      part[0][vi][vrow] = s;
      __syncthreads();
      s = vi == 0 ? (part[0][0][vrow] + part[0][1][vrow]) + (part[0][2][vrow] + part[0][3][vrow]) : 0.f;
    }
    store_largest(s, sizes + 2 * sizes_of_out + (((long long)bv * a.G + hk) * blocks_v + block_v) * 8);
  }
}

// dtable[n,h] = the head's sums over the relative positions of bucket n; one block each, in a fixed order: lanes along as many
// positions as the bucket has, up to 32, and along rows of sums beside that.  Latency: 5 us for 64 rows and 32 buckets of 16 heads (B=8,
// L=512), 8.6 for 128 rows whose buckets reach 472 positions (B=2, L=4096; 11 with 256 threads).
__global__ void __launch_bounds__(512)
table_finish_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Starts st, const float* partial, int rows, int reach,
                    sb_half* out, long long sN, long long sH) {
  __shared__ float part[16];
  grid_dependency_sync();
  const int n = blockIdx.x, h = blockIdx.y, entries = 2 * reach + 1;
  const bool behind = n >= a.n;
  const int i = behind ? n - a.n : n;
  // distances lo .. hi; without `bidirectional` every key behind the query has distance 0
  const int lo = behind ? max(st.s[i], 1) : st.s[i], hi = i + 1 < a.n ? min(st.s[i + 1] - 1, reach) : reach;
  const int from = behind ? reach + lo : reach - hi;
  const int to = behind ? reach + hi : !a.bidirectional && lo == 0 && hi >= 0 ? 2 * reach : reach - lo;
  const int run = to - from + 1;
  int across = 1;
  while (across < run && across < 32) across *= 2;
  const int lane = threadIdx.x & 31, each = 32 / across, r0 = (threadIdx.x >> 5) * each + lane / across;
  const float* base = partial + (long long)h * rows * entries + from;
  float s = 0.f;
  for (int c = lane % across; c < run; c += across)
#pragma unroll 8
    for (int r = r0; r < rows; r += 16 * each) s += base[(long long)r * entries + c];
  s = group_sum<32>(s);
  if (lane == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = group_sum<16>(part[threadIdx.x & 15]);
    if (threadIdx.x == 0) out[n * sN + h * sH] = sb_f2h(s);
  }
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
// Scratch: rows of biases, a packed copy of each operand that tensor maps cannot address, the work queue's counter.
struct Plan { int pitch, reach; size_t at[4], next, bytes; };
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
  p.next = p.bytes;
  p.bytes += 256;
  return p;
}
// x becomes a copy at `at`, which launch_pack() makes.
void pack(PackJobs* jobs, void* scratch, size_t at, Proj* x) {
  const int Pp = (x->P + 7) / 8 * 8;
  auto mag = [](long long v) { return v < 0 ? -v : v; };
  auto& j = jobs->job[jobs->n++];
  j.x = *x;
  j.dst = reinterpret_cast<sb_half*>(reinterpret_cast<char*>(scratch) + at);
  j.first = jobs->blocks;
  j.mode = x->sR == 1 && x->R % 2 == 0 && !((x->sP | x->sH | x->sB) & 1) && !(reinterpret_cast<uintptr_t>(x->p) & 3u) ? kPackTwos
           : x->R > 1 && mag(x->sR) < mag(x->sP) ? kPackRows : kPackFeatures;
  jobs->blocks += x->H * x->B * ((x->R + 63) / 64);
  x->p = j.dst;
  x->sP = 1; x->sR = Pp; x->sH = (long long)Pp * x->R; x->sB = x->sH * x->H;
}
int launch_pack(cudaStream_t s, const PackJobs& jobs) {
  if (jobs.n > 0) SB_LAUNCH_OK(launch_k(pack_rows_kernel, (unsigned)jobs.blocks, 256, 0, s, jobs));
  return SB_OK;
}
// Copies what tensor maps cannot address.
int pack_indirect(cudaStream_t s, void* scratch, const size_t* at, std::initializer_list<Proj*> operands) {
  PackJobs jobs;
  memset(&jobs, 0, sizeof(jobs));
  for (Proj* x : operands) {
    if (!rel_direct(*x)) pack(&jobs, scratch, *at, x);
    ++at;
  }
  return launch_pack(s, jobs);
}
Expand expansion(void* scratch, const Plan& pl) {
  return {reinterpret_cast<float*>(scratch), pl.pitch, pl.reach, reinterpret_cast<int*>(reinterpret_cast<char*>(scratch) + pl.next)};
}
RelTables tables_of(const Expand& x) { return {x.rows, x.pitch, x.reach}; }

}  // namespace

namespace {

// Rows in 16-byte pieces, any strides between them.
bool piecewise(const Proj& x) {
  auto ok = [](long long n, long long stride) { return n == 1 || stride % 8 == 0; };
  return (x.sP == 1 || x.P == 1) && !(reinterpret_cast<uintptr_t>(x.p) & 15u) && ok(x.H, x.sH) && ok(x.B, x.sB) && ok(x.R, x.sR);
}

// The forward pass with few queries: how many shares the keys are cut into, 0 when the tile kernel is to run.  The tile kernel has an
// item for 128 queries of one head, which walks the keys alone at 0.7 us per 64 of them; here 16 rows of all heads that share keys
// walk as many shares of the keys as there is room for.  So they are few when their CTAs do not fill the SMs and there are keys to
// share out (8 heads of 64, 256 queries, 4096 keys: 27 against 54 us here; 64 queries and keys: 8.2 against 7.2), and beyond that
// when there are not more CTAs than items: every key is read as often (64 x 16 heads, one query, 512 keys: 38 against 41 us), with
// heads that share keys less often (64 x 16 heads on 8, 4096 keys: 84 against 225); with more than four queries the tensor cores
// of the tile kernel outweigh that (16 queries, 512 keys: 52 against 41).
// The device's SMs count here and not the budget of sb_set_sm_budget: the number of shares is an order of summation, and results do not
// depend on the budget.  (Its CTAs are many short ones, which make room for another kernel's as they end.)
int few_splits(const Proj& q, const Proj& k) {
  const long long sms = device_facts().sms;
  const long long blocks = ((long long)(q.H / k.H) * q.R + 15) / 16, ctas = blocks * k.B * k.H, items = (long long)q.B * q.H * ((q.R + 127) / 128);
  const bool idle = ctas <= sms && (blocks == 1 || k.R >= 1024);
  if (!idle && ctas * (q.R > 4 ? 2 : 1) > items) return 0;
  // two CTAs for each SM and no more, which would wait for those (B=16, 16 heads on 8, 8192 keys of 128 features, 128 CTAs: two
  // shares 87 us, four 97, five 114), at least 256 keys a share
  return (int)std::max<long long>(1, std::min<long long>({2 * sms / ctas, (k.R + 255) / 256, 64}));
}
struct FewPlan { int splits; size_t k, v, bytes; };
FewPlan few_plan(const Proj& q, const Proj& k, const Proj& v) {
  FewPlan f;
  f.splits = few_splits(q, k);
  f.bytes = f.splits > 1 ? align256(sizeof(float) * (size_t)q.H * q.B * q.R * f.splits * ((q.P <= 64 ? 64 : 128) + 2)) : 0;
  f.k = f.bytes;
  if (!piecewise(k)) f.bytes += packed_bytes(k);
  f.v = f.bytes;
  if (!piecewise(v)) f.bytes += packed_bytes(v);
  return f;
}

template <int P>
int launch_few(cudaStream_t s, FewParams& p, const Starts& st) {
  const int share = share_of(p.a.K, p.splits);
  p.slots = FewCfg<P>::slots(share);
  SB_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(few_queries_kernel<P>), FewCfg<P>::smem(1 << 30)));
  const long long units = (long long)p.a.B * p.a.G;
  SB_LAUNCH_OK(launch_k(few_queries_kernel<P>, (unsigned)(units * p.blocks * p.splits), kFewThreads, FewCfg<P>::smem(share), s, p, st));
  if (p.splits > 1)
    SB_LAUNCH_OK(launch_k(join_splits_kernel<P>, (unsigned)((units * p.rows + 3) / 4), 128, 0, s, p));
  return SB_OK;
}

}  // namespace

size_t rel_attn_scratch_bytes(const Proj& q, const Proj& k, const Proj& v, const RelBias& bias) {
  return few_splits(q, k) ? few_plan(q, k, v).bytes : plan_of({&q, &k, &v}, q.H, bias).bytes;
}

int launch_rel_attn_fwd(cudaStream_t s, void* scratch, Proj q, Proj k, Proj v, const RelBias& bias, Proj out, RelRows lse, const RelSpan& span) {
  Starts st;
  AttnArgs a = attn_args(q, k, v, bias, out, lse, span, &st);
  if (few_splits(q, k)) {
    const FewPlan f = few_plan(q, k, v);
    PackJobs jobs;
    memset(&jobs, 0, sizeof(jobs));
    if (!piecewise(k)) pack(&jobs, scratch, f.k, &k);
    if (!piecewise(v)) pack(&jobs, scratch, f.v, &v);
    SB_TRY(launch_pack(s, jobs));
    FewParams p;
    a.k = k; a.v = v;
    p.a = a;
    p.rows = (q.H / k.H) * q.R;
    p.blocks = (p.rows + 15) / 16;
    p.splits = f.splits;
    p.reach = std::max(1, bias.starts[bias.n - 1]);
    p.before = bias.n - 1;
    p.behind = 0;
    if (bias.bidirectional) p.behind = 2 * bias.n - 1;
    else while (p.behind + 1 < bias.n && bias.starts[p.behind + 1] <= 0) ++p.behind;
    p.partial = f.splits > 1 ? reinterpret_cast<float*>(scratch) : nullptr;
    return q.P <= 64 ? launch_few<64>(s, p, st) : launch_few<128>(s, p, st);
  }
  const Plan pl = plan_of({&q, &k, &v}, q.H, bias);
  const Expand x = expansion(scratch, pl);
  SB_LAUNCH_OK(launch_k(expand_bias_kernel, dim3(expand_blocks(x.pitch), a.H), 256, 0, s, a, st, x));
  SB_TRY(pack_indirect(s, scratch, pl.at, {&q, &k, &v}));
  return launch_rel_tiles_fwd(s, q, k, v, tables_of(x), x.next, out, lse, span);
}

namespace {
// and for the backward pass records and sums
struct BwdPlan { Plan p; size_t records, sizes, partial, bytes; int rows; };
BwdPlan bwd_plan(const Proj& dout, const Proj& q, const Proj& k, const Proj& v, const RelBias& bias) {
  BwdPlan b;
  b.p = plan_of({&dout, &q, &k, &v}, q.H, bias);
  b.rows = q.B * ((q.R + 127) / 128) * 2;
  b.records = b.p.bytes;
  const size_t blocks = (size_t)q.H * q.B * ((q.R + 63) / 64), blocks_v = (size_t)v.H * v.B * ((v.R + 63) / 64);
  b.sizes = b.records + align256(sizeof(float) * 192 * blocks);
  b.partial = b.sizes + (kRelScaled ? align256(sizeof(float) * 8 * (2 * blocks + blocks_v)) : 0);
  b.bytes = b.partial + align256(sizeof(float) * (size_t)q.H * b.rows * (2 * b.p.reach + 1));
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
  const Expand x = expansion(scratch, pl.p);
  auto pieces = [](const Proj& x) {
    return x.sP == 1 && x.P % 8 == 0 && !((x.sH | x.sB | x.sR) & 7) && !(reinterpret_cast<uintptr_t>(x.p) & 15u);
  };
  float* records = reinterpret_cast<float*>(base + pl.records);
  float* sizes = reinterpret_cast<float*>(base + pl.sizes);
  const int expanding = a.H * expand_blocks(x.pitch), values = kRelScaled && !rel_both(q, k) ? a.G * a.B * ((a.K + 63) / 64) : 0;
  auto kernel = values ? (q.P <= 64 ? row_records_kernel<64, kRelScaled> : row_records_kernel<128, kRelScaled>)
                       : (q.P <= 64 ? row_records_kernel<64, false> : row_records_kernel<128, false>);
  const int rows = a.H * a.B * ((a.J + 63) / 64);
  SB_LAUNCH_OK(launch_k(kernel, (unsigned)(expanding + std::max(rows, values)), 256, 0, s, a, st, x, records, sizes,
                        pieces(dout) && pieces(out) ? 1 : 0, pieces(v) ? 1 : 0, expanding, rows, values));
  SB_TRY(pack_indirect(s, scratch, pl.p.at, {&dout, &q, &k, &v}));
  float* partial = reinterpret_cast<float*>(base + pl.partial);
  SB_TRY(launch_rel_tiles_bwd(s, dout, q, k, v, tables_of(x), RelBackward{records, sizes, partial, x.next}, dq, dk, dv, span));
  SB_LAUNCH_OK(launch_k(table_finish_kernel, dim3(a.buckets, a.H), 512, 0, s, a, st, partial, pl.rows, pl.p.reach,
                        reinterpret_cast<sb_half*>(dtable), dt_sN, dt_sH));
  return SB_OK;
}

}  // namespace sb
