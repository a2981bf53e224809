// Attention with a sliding window and a few first tokens that stay visible (sinks), head dims
// 32 / 64 / 128, key-padding mask, grouped key/value heads, forward and backward.
//
//   key j is visible to query i   iff   mask[j]  and  j <= i + right  and  (j >= i - left  or  j < sinks)
//   p_ij = exp(scale q_i.k_j - m_i) / l_i over the visible keys,  o_i = sum_j p_ij v_j
//   a query without a visible key has o = 0 and contributes no gradient
//   D_i = do_i.o_i,  dS_ij = p_ij (do_i.v_j - D_i),  dq_i = scale sum_j dS_ij k_j,
//   dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i p_ij do_i
//
// Work per (query, key) pair is the same as in dense attention, but only the key tiles that hold a
// visible pair are read: O(L (left + right + sinks)) instead of O(L^2).  A tile is 64 rows staged
// in LDS; a wave owns 32 rows of the other side in registers and walks the tile in 32 x 32
// blocks, each of which is empty (skipped), full (no mask arithmetic) or partial (one 32-bit
// visibility word per lane) — all three decided by scalar arithmetic on the block's corners.
//
// Products run on v_mfma_f32_32x32x16_bf16 in the transposed orientation: the lane's column is
// the row it owns, so the softmax statistics are lane-local (plus one exchange between the two
// half-waves) and the accumulator registers, rounded to bf16, are directly the B operand of the
// next product; its A operand is the transpose of a row-major LDS tile, by ds_read_b64_tr_b16.
//
// Accumulators, softmax statistics, D and the log-sum-exp are fp32.  P and dS are rounded to bf16
// (half a step, at most 2^-8 relative) because the matrix unit's operands are bf16; the row sum l adds
// the unrounded values.  No atomics: every output element has one writer and one order of sums.
#include "common.h"

namespace pv {
namespace wattn {

constexpr int TK = 64;   // rows per staged tile
constexpr int NTH = 256;
constexpr int RB = 128;  // rows a workgroup owns: 4 waves x 32
constexpr float LOG2E = 1.4426950408889634f;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// element strides of a (N, L, heads, d) operand whose last dimension is contiguous
struct View {
  unsigned short* p;
  long n, l, h;
};

struct Args {
  View q, k, v, o, go, dq, dk, dv;
  const void* mask;  // (N, L), mask_bytes 1 or 4, rows mask_n elements apart; null: all keys
  long mask_n;
  int mask_bytes;
  float* lse;  // (N, H, L), log2 domain, includes the scale; null: not kept
  float* dd;   // (N, H, L)  D
  int L, H, G;  // G = query heads per key/value head
  int left, right, sinks;
  float scale;
  int tiles;  // ceil(L / RB)
};

#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16((a), (b), (c), 0, 0, 0)

__device__ __forceinline__ int mask_at(const Args& a, int n, int r) {
  const long i = (long)n * a.mask_n + r;
  return a.mask_bytes == 1 ? (int)reinterpret_cast<const unsigned char*>(a.mask)[i]
                           : reinterpret_cast<const int*>(a.mask)[i];
}

// Registers of a tile on its way to LDS: D / 32 16-byte pieces per thread.  Rows behind the
// sequence and masked rows are stored as zeros, so whatever they hold (infinities and NaN
// too) never meets a zero probability in a product.
template <int D>
struct Stage {
  u32x4 v[D / 32];
};

template <int D>
__device__ __forceinline__ void tile_load(const unsigned short* base, long ls, int r0, int L, Stage<D>& s) {
#pragma unroll
  for (int u = 0; u < D / 32; ++u) {
    const int c = threadIdx.x + NTH * u;
    const int r = c / (D / 8), e = (c % (D / 8)) * 8;
    s.v[u] = *reinterpret_cast<const u32x4*>(base + (long)min(r0 + r, L - 1) * ls + e);
  }
}

template <int D>
__device__ __forceinline__ void tile_store(unsigned short* t, const Stage<D>& s, unsigned long long keep) {
#pragma unroll
  for (int u = 0; u < D / 32; ++u) {
    const int c = threadIdx.x + NTH * u;
    const int r = c / (D / 8), e = (c % (D / 8)) * 8;
    const bool ok = (keep >> r) & 1ull;
    *reinterpret_cast<u32x4*>(t + r * (D + 8) + e) = ok ? s.v[u] : u32x4{0, 0, 0, 0};
  }
}

// bits of the tile's rows that exist and are not masked (every wave computes the same word)
__device__ __forceinline__ unsigned long long tile_keep(const Args& a, int n, int r0) {
  const int r = r0 + (threadIdx.x & 63);
  bool ok = r < a.L;
  if (ok && a.mask) ok = mask_at(a, n, r) != 0;
  return __ballot(ok);
}

// A operand: rows r0 .. r0+31 of a tile, columns 16 s + 8 (lane / 32) ..
template <int D>
__device__ __forceinline__ bf16x8 row_frag(const unsigned short* t, int r0, int s) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const bf16x8*>(t + (r0 + (lane & 31)) * (D + 8) + s * 16 + (lane >> 5) * 8);
}

// A operand, transposed: row = tile column c0 + (lane & 31); its 8 k-slots are the tile rows that a
// 32 x 32 accumulator's registers 8 s .. 8 s + 7 hold in this half-wave: r0 + 16 s + 4 h + {0..3}, +8
template <int D>
__device__ __forceinline__ bf16x8 tr_frag(const unsigned short* t, int r0, int s, int c0) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const unsigned short* p =
      t + (r0 + 16 * s + 4 * (g >> 1) + ((lane & 15) >> 2)) * (D + 8) + c0 + 16 * (g & 1) + 4 * (lane & 3);
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 8 * (D + 8)));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// B operand: this lane's row of a global matrix, columns 16 s + 8 (lane / 32) ..; zeros if !ok
template <int D>
__device__ __forceinline__ void glob_frag(const unsigned short* row, bool ok, bf16x8 (&f)[D / 16]) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
    f[s] = ok ? *reinterpret_cast<const bf16x8*>(row + s * 16 + h * 8) : bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& x, int s) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[8 * s + 2 * i], x[8 * s + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, w);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// accumulator register r of half-wave h holds row (r & 3) + 8 (r >> 2) + 4 h
__device__ __forceinline__ constexpr int reg_bit(int r) { return (r & 3) + 8 * (r >> 2); }

// bits lo .. hi of a word (lo, hi any integers)
__device__ __forceinline__ unsigned bits_between(int lo, int hi) {
  const unsigned up = hi >= 31 ? 0xFFFFFFFFu : hi < 0 ? 0u : (2u << hi) - 1u;
  const unsigned dn = lo <= 0 ? 0xFFFFFFFFu : lo > 31 ? 0u : ~((1u << lo) - 1u);
  return up & dn;
}

enum { EMPTY = 0, PARTIAL = 1, FULL = 2 };

// 32 queries i0 .. i0+31 against 32 keys j0 .. j0+31, kw = the keys' keep bits; uniform arguments
__device__ __forceinline__ int block_kind(const Args& a, int i0, int j0, unsigned kw) {
  if (kw == 0u || j0 > i0 + 31 + a.right) return EMPTY;
  if (j0 + 31 < i0 - a.left && j0 >= a.sinks) return EMPTY;
  const bool low = j0 >= i0 + 31 - a.left || j0 + 31 < a.sinks;
  return (kw == 0xFFFFFFFFu && low && j0 + 31 <= i0 + a.right) ? FULL : PARTIAL;
}

// the keys of j0 .. j0+31 that query i sees, as bits
__device__ __forceinline__ unsigned seen_keys(const Args& a, int i, int j0, unsigned kw) {
  return kw & (bits_between(i - a.left - j0, i + a.right - j0) |
               (bits_between(0, a.sinks - 1 - j0) & bits_between(0, i + a.right - j0)));
}

// key tiles of the queries i0 .. i1: `sink` tiles from 0, then lo .. hi
struct Walk {
  int sink, lo, n;
  __device__ __forceinline__ int tile(int it) const { return it < sink ? it : lo + it - sink; }
};
__device__ __forceinline__ Walk key_walk(const Args& a, int i0, int i1) {
  Walk w;
  w.lo = max(0, i0 - a.left) / TK;
  const int hi = min(a.L - 1, i1 + a.right) / TK;
  w.sink = min((a.sinks + TK - 1) / TK, w.lo);
  w.n = w.sink + hi - w.lo + 1;
  return w;
}

// ------------------------------------------------------------------------------------ forward
// Workgroup = 128 queries of one head; a wave owns 32 of them (lane & 31), both half-waves hold the
// same queries and split the keys of each block.
template <int D>
__global__ __launch_bounds__(NTH, 2) void fwd_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) unsigned short kt[2][TK * (D + 8)];
  __shared__ __attribute__((aligned(16))) unsigned short vt[2][TK * (D + 8)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = bid % a.tiles, nh = bid / a.tiles;
  const int hd = nh % a.H, n = nh / a.H, kvh = hd / a.G;
  const int b0 = tile * RB, w0 = b0 + wave * 32, i = w0 + (lane & 31);
  const unsigned short* K = a.k.p + n * a.k.n + kvh * a.k.h;
  const unsigned short* V = a.v.p + n * a.v.n + kvh * a.v.h;
  const float sl = a.scale * LOG2E;
  bf16x8 qf[D / 16];
  glob_frag<D>(a.q.p + n * a.q.n + (long)min(i, a.L - 1) * a.q.l + hd * a.q.h, i < a.L, qf);
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c] = zero16();
  float m = -INFINITY, l = 0.f;
  const Walk wk = key_walk(a, b0, min(b0 + RB, a.L) - 1);
  Stage<D> sk, sv;
  int t0 = wk.tile(0) * TK;
  tile_load<D>(K, a.k.l, t0, a.L, sk);
  tile_load<D>(V, a.v.l, t0, a.L, sv);
  unsigned long long keep = tile_keep(a, n, t0);
  tile_store<D>(kt[0], sk, keep);
  tile_store<D>(vt[0], sv, keep);
  __syncthreads();
  int buf = 0;
  for (int it = 0; it < wk.n; ++it, buf ^= 1) {
    const int j0 = t0;
    const unsigned long long kw = keep;
    if (it + 1 < wk.n) {
      t0 = wk.tile(it + 1) * TK;
      tile_load<D>(K, a.k.l, t0, a.L, sk);
      tile_load<D>(V, a.v.l, t0, a.L, sv);
      keep = tile_keep(a, n, t0);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int jb = j0 + 32 * c;
      const unsigned kwc = (unsigned)(kw >> (32 * c));
      const int kind = w0 < a.L ? block_kind(a, w0, jb, kwc) : EMPTY;
      if (kind == EMPTY) continue;
      f32x16 s = zero16();
#pragma unroll
      for (int t = 0; t < D / 16; ++t) s = MFMA32(row_frag<D>(kt[buf], 32 * c, t), qf[t], s);
      if (kind == PARTIAL) {
        const unsigned see = seen_keys(a, i, jb, kwc) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (see >> reg_bit(r)) & 1u ? s[r] : -INFINITY;
      }
      float bm = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[r]);
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      const float mn = fmaxf(m, bm);
      const float ms = mn == -INFINITY ? 0.f : mn * sl;
      if (__ballot(mn > m) != 0ull) {
        const float corr = __builtin_amdgcn_exp2f(fmaf(m, sl, -ms));  // 0 at the first visible key
        l *= corr;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] *= corr;
        m = mn;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl, -ms));
        l += s[r];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 pb = pack8(s, t);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = MFMA32(tr_frag<D>(vt[buf], 32 * c, t, 32 * e), pb, o[e]);
      }
    }
    if (it + 1 < wk.n) {
      tile_store<D>(kt[buf ^ 1], sk, keep);
      tile_store<D>(vt[buf ^ 1], sv, keep);
    }
    __syncthreads();
  }
  l += __shfl_xor(l, 32, 64);
  if (i >= a.L) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
  unsigned short* orow = a.o.p + n * a.o.n + (long)i * a.o.l + hd * a.o.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; ++t)
      *reinterpret_cast<uint2*>(orow + e * 32 + 8 * t + 4 * h) =
          uint2{pack_bf16x2(o[e][4 * t] * inv, o[e][4 * t + 1] * inv),
                pack_bf16x2(o[e][4 * t + 2] * inv, o[e][4 * t + 3] * inv)};
  if (a.lse && h == 0)
    a.lse[((long)n * a.H + hd) * a.L + i] = l == 0.f ? INFINITY : fmaf(m, sl, __log2f(l));
}

// ------------------------------------------------------------------------------------ backward: dq, D
// Same walk as the forward: dS^T in registers, dq^T += K^T dS^T.  D is the lane's own row sum of
// do * o and goes to memory for the other kernel.
template <int D>
__global__ __launch_bounds__(NTH, D <= 64 ? 2 : 1) void bwd_dq_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) unsigned short kt[2][TK * (D + 8)];
  __shared__ __attribute__((aligned(16))) unsigned short vt[2][TK * (D + 8)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = bid % a.tiles, nh = bid / a.tiles;
  const int hd = nh % a.H, n = nh / a.H, kvh = hd / a.G;
  const int b0 = tile * RB, w0 = b0 + wave * 32, i = w0 + (lane & 31), ic = min(i, a.L - 1);
  const unsigned short* K = a.k.p + n * a.k.n + kvh * a.k.h;
  const unsigned short* V = a.v.p + n * a.v.n + kvh * a.v.h;
  const float sl = a.scale * LOG2E;
  bf16x8 qf[D / 16], gf[D / 16];
  glob_frag<D>(a.q.p + n * a.q.n + (long)ic * a.q.l + hd * a.q.h, i < a.L, qf);
  glob_frag<D>(a.go.p + n * a.go.n + (long)ic * a.go.l + hd * a.go.h, i < a.L, gf);
  float dd = 0.f;
  {
    bf16x8 of[D / 16];
    glob_frag<D>(a.o.p + n * a.o.n + (long)ic * a.o.l + hd * a.o.h, i < a.L, of);
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        dd = fmaf(bf16_to_f32((unsigned short)of[s][e]), bf16_to_f32((unsigned short)gf[s][e]), dd);
  }
  dd += __shfl_xor(dd, 32, 64);
  const long row = ((long)n * a.H + hd) * a.L + ic;
  const float lse = a.lse[row];
  if (i < a.L && h == 0) a.dd[row] = dd;
  f32x16 acc[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc[c] = zero16();
  const Walk wk = key_walk(a, b0, min(b0 + RB, a.L) - 1);
  Stage<D> sk, sv;
  int t0 = wk.tile(0) * TK;
  tile_load<D>(K, a.k.l, t0, a.L, sk);
  tile_load<D>(V, a.v.l, t0, a.L, sv);
  unsigned long long keep = tile_keep(a, n, t0);
  tile_store<D>(kt[0], sk, keep);
  tile_store<D>(vt[0], sv, keep);
  __syncthreads();
  int buf = 0;
  for (int it = 0; it < wk.n; ++it, buf ^= 1) {
    const int j0 = t0;
    const unsigned long long kw = keep;
    if (it + 1 < wk.n) {
      t0 = wk.tile(it + 1) * TK;
      tile_load<D>(K, a.k.l, t0, a.L, sk);
      tile_load<D>(V, a.v.l, t0, a.L, sv);
      keep = tile_keep(a, n, t0);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int jb = j0 + 32 * c;
      const unsigned kwc = (unsigned)(kw >> (32 * c));
      const int kind = w0 < a.L ? block_kind(a, w0, jb, kwc) : EMPTY;
      if (kind == EMPTY) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        s = MFMA32(row_frag<D>(kt[buf], 32 * c, t), qf[t], s);
        dp = MFMA32(row_frag<D>(vt[buf], 32 * c, t), gf[t], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl, -lse)) * (dp[r] - dd);
      if (kind == PARTIAL) {
        const unsigned see = seen_keys(a, i, jb, kwc) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (see >> reg_bit(r)) & 1u ? s[r] : 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 b = pack8(s, t);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = MFMA32(tr_frag<D>(kt[buf], 32 * c, t, 32 * e), b, acc[e]);
      }
    }
    if (it + 1 < wk.n) {
      tile_store<D>(kt[buf ^ 1], sk, keep);
      tile_store<D>(vt[buf ^ 1], sv, keep);
    }
    __syncthreads();
  }
  if (i >= a.L) return;
  unsigned short* drow = a.dq.p + n * a.dq.n + (long)i * a.dq.l + hd * a.dq.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; ++t)
      *reinterpret_cast<uint2*>(drow + e * 32 + 8 * t + 4 * h) =
          uint2{pack_bf16x2(acc[e][4 * t] * a.scale, acc[e][4 * t + 1] * a.scale),
                pack_bf16x2(acc[e][4 * t + 2] * a.scale, acc[e][4 * t + 3] * a.scale)};
}

// ------------------------------------------------------------------------------------ backward: dk, dv
// Workgroup = 128 keys of one key/value head, a wave owns 32 of them; it walks the query tiles of
// every query head of the group: P and dS (queries x keys), dv^T += dO^T P, dk^T += Q^T dS.
template <int D>
__global__ __launch_bounds__(NTH, D <= 64 ? 2 : 1) void bwd_dkv_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) unsigned short qt[2][TK * (D + 8)];
  __shared__ __attribute__((aligned(16))) unsigned short gt[2][TK * (D + 8)];
  __shared__ __attribute__((aligned(16))) float ls[2][TK], ds[2][TK];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int Hkv = a.H / a.G;
  const int tile = bid % a.tiles, nh = bid / a.tiles;
  const int kvh = nh % Hkv, n = nh / Hkv;
  const int b0 = tile * RB, w0 = b0 + wave * 32, j = w0 + (lane & 31), jc = min(j, a.L - 1);
  const float sl = a.scale * LOG2E;
  bool ok = j < a.L;
  if (ok && a.mask) ok = mask_at(a, n, j) != 0;
  const bool all_ok = (__ballot(ok) == ~0ull), any_ok = (__ballot(ok) != 0ull);
  bf16x8 kf[D / 16], vf[D / 16];
  glob_frag<D>(a.k.p + n * a.k.n + (long)jc * a.k.l + kvh * a.k.h, ok, kf);
  glob_frag<D>(a.v.p + n * a.v.n + (long)jc * a.v.l + kvh * a.v.h, ok, vf);
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = zero16();
  // queries that see a key of this workgroup: from b0 - right to the last key + left, or to the
  // end where the workgroup holds sinks
  const int lo = max(0, b0 - a.right) / TK;
  const int last = b0 < a.sinks ? a.L - 1 : min(a.L - 1, min(b0 + RB, a.L) - 1 + a.left);
  const int per = last / TK - lo + 1, total = per * a.G;
  Stage<D> sq, sg;
  float sls = 0.f, sds = 0.f;
  auto load = [&](int it) {
    const int hd = kvh * a.G + it / per, r0 = (lo + it % per) * TK;
    tile_load<D>(a.q.p + n * a.q.n + hd * a.q.h, a.q.l, r0, a.L, sq);
    tile_load<D>(a.go.p + n * a.go.n + hd * a.go.h, a.go.l, r0, a.L, sg);
    if (threadIdx.x < TK) {
      const long row = ((long)n * a.H + hd) * a.L + min(r0 + (int)threadIdx.x, a.L - 1);
      sls = a.lse[row];
      sds = a.dd[row];
    }
  };
  auto store = [&](int it, int b) {
    const int r0 = (lo + it % per) * TK;
    const unsigned long long keep = a.L - r0 >= 64 ? ~0ull : (1ull << (a.L - r0)) - 1ull;
    tile_store<D>(qt[b], sq, keep);
    tile_store<D>(gt[b], sg, keep);
    if (threadIdx.x < TK) {
      ls[b][threadIdx.x] = sls;
      ds[b][threadIdx.x] = sds;
    }
  };
  load(0);
  store(0, 0);
  __syncthreads();
  int buf = 0;
  for (int it = 0; it < total; ++it, buf ^= 1) {
    const int r0 = (lo + it % per) * TK;
    if (it + 1 < total) load(it + 1);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i0 = r0 + 32 * c;
      // the same three kinds as in the forward, seen from the keys
      if (!any_ok || i0 >= a.L || i0 + 31 < w0 - a.right || (i0 > w0 + 31 + a.left && w0 >= a.sinks)) continue;
      const bool full = all_ok && i0 + 31 < a.L && i0 >= w0 + 31 - a.right &&
                        (i0 + 31 <= w0 + a.left || w0 + 31 < a.sinks);
      f32x16 p = zero16(), dp = zero16();
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        p = MFMA32(row_frag<D>(qt[buf], 32 * c, t), kf[t], p);
        dp = MFMA32(row_frag<D>(gt[buf], 32 * c, t), vf[t], dp);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 lv = *reinterpret_cast<const f32x4*>(&ls[buf][32 * c + 8 * t + 4 * h]);
        const f32x4 dv4 = *reinterpret_cast<const f32x4*>(&ds[buf][32 * c + 8 * t + 4 * h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * t + e;
          p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], sl, -lv[e]));
          dp[r] = p[r] * (dp[r] - dv4[e]);
        }
      }
      if (!full) {
        const int hi = min(a.L - 1, j < a.sinks ? a.L - 1 : j + a.left);
        const unsigned see = (ok ? bits_between(j - a.right - i0, hi - i0) : 0u) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool s = (see >> reg_bit(r)) & 1u;
          p[r] = s ? p[r] : 0.f;
          dp[r] = s ? dp[r] : 0.f;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 pb = pack8(p, t), sb = pack8(dp, t);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          dv[e] = MFMA32(tr_frag<D>(gt[buf], 32 * c, t, 32 * e), pb, dv[e]);
          dk[e] = MFMA32(tr_frag<D>(qt[buf], 32 * c, t, 32 * e), sb, dk[e]);
        }
      }
    }
    if (it + 1 < total) store(it + 1, buf ^ 1);
    __syncthreads();
  }
  if (j >= a.L) return;
  unsigned short* kr = a.dk.p + n * a.dk.n + (long)j * a.dk.l + kvh * a.dk.h;
  unsigned short* vr = a.dv.p + n * a.dv.n + (long)j * a.dv.l + kvh * a.dv.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      *reinterpret_cast<uint2*>(kr + e * 32 + 8 * t + 4 * h) =
          uint2{pack_bf16x2(dk[e][4 * t] * a.scale, dk[e][4 * t + 1] * a.scale),
                pack_bf16x2(dk[e][4 * t + 2] * a.scale, dk[e][4 * t + 3] * a.scale)};
      *reinterpret_cast<uint2*>(vr + e * 32 + 8 * t + 4 * h) =
          uint2{pack_bf16x2(dv[e][4 * t], dv[e][4 * t + 1]), pack_bf16x2(dv[e][4 * t + 2], dv[e][4 * t + 3])};
    }
}

#undef MFMA32

// operand i of a call: pointer and its three element strides st[3 i ..]
__host__ inline View view(const void* p, const long* st, int i) {
  return View{(unsigned short*)const_cast<void*>(p), st[3 * i], st[3 * i + 1], st[3 * i + 2]};
}

// sizes that the kernels' 32-bit row arithmetic and their 1-D grids hold
__host__ inline int check_sizes(long N, long L, long H, long G, int d, float scale) {
  if (N <= 0 || L <= 0 || H <= 0 || G <= 0 || H % G) return -1;
  if (d != 32 && d != 64 && d != 128) return -2;
  if (L > (1L << 29) || !(scale > 0.f)) return -3;
  const long blocks = (L + RB - 1) / RB * H * N;
  return blocks > 0x7FFFFFFFL ? -4 : 0;
}

}  // namespace wattn
}  // namespace pv

using namespace pv;
using namespace pv::wattn;

namespace {
Args common(const void* q, const void* k, const void* v, const void* o, const long* st, const void* mask, long mask_n,
            int mask_bytes, float* lse, int L, int H, int G, int left, int right, int sinks, float scale) {
  Args a{};
  a.q = view(q, st, 0);
  a.k = view(k, st, 1);
  a.v = view(v, st, 2);
  a.o = view(o, st, 3);
  a.mask = mask;
  a.mask_n = mask_n;
  a.mask_bytes = mask_bytes;
  a.lse = lse;
  a.L = L, a.H = H, a.G = G;
  a.left = min(left, L), a.right = min(right, L), a.sinks = min(sinks, L);
  a.scale = scale;
  a.tiles = (L + RB - 1) / RB;
  return a;
}
}  // namespace

// q, o (N, L, H, d), k, v (N, L, H / G, d) bf16; st: element strides {n, l, h} of q, k, v, o
// (multiples of 8, 16-byte aligned pointers); left, right >= L: unbounded.  lse (N, H, L) fp32 or null.
PV_API int pv_wattn_fwd(const void* q, const void* k, const void* v, void* o, const long* st, const void* mask,
                        long mask_n, int mask_bytes, float* lse, int N, int L, int H, int G, int d, int left,
                        int right, int sinks, float scale, void* stream) {
  if (const int rc = check_sizes(N, L, H, G, d, scale)) return rc;
  const Args a = common(q, k, v, o, st, mask, mask_n, mask_bytes, lse, L, H, G, left, right, sinks, scale);
  const dim3 grid((unsigned)((long)a.tiles * H * N));
  if (d == 32) hipLaunchKernelGGL(fwd_kernel<32>, grid, dim3(NTH), 0, (hipStream_t)stream, a);
  else if (d == 64) hipLaunchKernelGGL(fwd_kernel<64>, grid, dim3(NTH), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(fwd_kernel<128>, grid, dim3(NTH), 0, (hipStream_t)stream, a);
  PV_LAUNCH_CHECK();
  return 0;
}

// st: strides of q, k, v, o, go, dq, dk, dv.  dd (N, H, L) fp32 workspace; dq (N, L, H, d), dk, dv
// (N, L, H / G, d) bf16, every element written.
PV_API int pv_wattn_bwd(const void* q, const void* k, const void* v, const void* o, const void* go, void* dq, void* dk,
                        void* dv, const long* st, const void* mask, long mask_n, int mask_bytes, float* lse, float* dd,
                        int N, int L, int H, int G, int d, int left, int right, int sinks, float scale, void* stream) {
  if (const int rc = check_sizes(N, L, H, G, d, scale)) return rc;
  Args a = common(q, k, v, o, st, mask, mask_n, mask_bytes, lse, L, H, G, left, right, sinks, scale);
  a.go = view(go, st, 4);
  a.dq = view(dq, st, 5);
  a.dk = view(dk, st, 6);
  a.dv = view(dv, st, 7);
  a.dd = dd;
  const dim3 gq((unsigned)((long)a.tiles * H * N)), gk((unsigned)((long)a.tiles * (H / G) * N));
  hipStream_t s = (hipStream_t)stream;
#define PV_WBWD(DV)                                                 \
  do {                                                              \
    hipLaunchKernelGGL(bwd_dq_kernel<DV>, gq, dim3(NTH), 0, s, a);  \
    PV_LAUNCH_CHECK();                                              \
    hipLaunchKernelGGL(bwd_dkv_kernel<DV>, gk, dim3(NTH), 0, s, a); \
    PV_LAUNCH_CHECK();                                              \
  } while (0)
  if (d == 32) PV_WBWD(32);
  else if (d == 64) PV_WBWD(64);
  else PV_WBWD(128);
#undef PV_WBWD
  return 0;
}
