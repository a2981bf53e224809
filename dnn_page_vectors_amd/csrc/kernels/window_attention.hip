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
constexpr int RB = 128;  // rows a workgroup owns: 4 waves x 32 (sequences up to SHORT: 2 waves, all rows)
// Up to SHORT tokens: one tile, so a single buffer, and two waves: more workgroups at a time.  4096 x 32 tokens x 12 heads,
// forward / backward: 229 / 703 us instead of 306 / 877; 2048 x 64 tokens 201 / 645 instead of 206 / 673.
constexpr int SHORT = TK;
// Query tiles per workgroup of the sinks' far part (4: 454 us instead of 448 for forward and backward of 64 pages x
// 975 tokens x 12 heads, 755 instead of 739 for 4 x 4096 x 16 of 128).
constexpr int FAR = 16;
constexpr float LOG2E = 1.4426950408889634f;
// The running maximum is raised only when a score passes it by more than this (log2 units): until then
// probabilities may be as large as 2^8, which costs fp32 sums and bf16 roundings nothing, and the
// accumulators are not rescaled (32 of ~110 vector instructions per block at d = 64).
constexpr float SLACK = 8.f;

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
  float* lse;  // (N, H, L)  minus the log-sum-exp of a row's scores (log2 units, scale included); null: not kept
  float* dd;   // (N, H, L)  minus D
  unsigned char* rest;  // rest_at: the next 8 bits of o below its bf16 (signed); with lse
  int L, H, G;  // G = query heads per key/value head
  int left, right, sinks;
  float scale;
  int tiles;  // ceil(L / RB)
  // backward: the sinks' far queries (see bwd_dkv_kernel); far_chunks = 0: not split off
  float* part;
  long far_main;  // slots of the near parts
  int far_chunks, far_blocks, far_tile, far_wgs;  // far_wgs: workgroups per sequence and key/value head
};

// What rounding a float to bf16 hi left out, to 2^-8 of hi's last place: D = do.o is subtracted from do.v_j, and with
// the rounded o the gradients of a narrow window were off by 0.0029 of their size (norms), with these bits by
// 0.0025, of which 0.0024 is the rounding of dS and of the result.  One byte per element, 3 to 5 % of the time of forward
// and backward (32 pages x 2000 tokens x 12 heads: 631 -> 650 us).
__device__ __forceinline__ int rest_of(float x, unsigned hi) {
  const int r = (int)(__builtin_bit_cast(unsigned, x) - (hi << 16));
  return min(max((r + 128) >> 8, -128), 127);
}
// Laid out for the two kernels' lanes, (N, H, ceil(L / 32), d / 8, 32 rows, 8): each store and load of a wave covers
// 256 bytes in a row (in o's own
// order, 8 bytes to a row at a time, forward and backward of the same pages took 666 us).
template <int D>
__device__ __forceinline__ unsigned char* rest_at(const Args& a, int n, int hd, int i, int eighth) {
  return a.rest + ((((long)n * a.H + hd) * ((a.L + 31) >> 5) + (i >> 5)) * (D / 8) + eighth) * 256 + (i & 31) * 8;
}
__device__ __forceinline__ float with_rest(unsigned short hi, int rest) {
  return __builtin_bit_cast(float, ((unsigned)hi << 16) + (unsigned)(rest << 8));
}

#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16((a), (b), (c), 0, 0, 0)

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- tiles in LDS ---------------------------------------------------------------------------
// [64 rows][D] bf16, rows of D / 8 16-byte chunks; chunk c of row r is stored at place c ^ swz(r), so that
// both the row reads (8 rows, one chunk each) and the transposed reads (4 rows, 4 chunks each)
// touch every bank once.
template <int D>
__device__ __forceinline__ constexpr int swz(int r) {
  return D == 32 ? ((r >> 2) & 1) << 1 : D == 64 ? (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1)
                                                 : ((r & 3) << 2) | (((r >> 2) & 1) << 1);
}

__device__ __forceinline__ unsigned lds_at(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<size_t>((__attribute__((address_space(3))) const char*)p));
}

// Tile rows go from memory straight to LDS (global_load_lds_dwordx4: 64 lanes x 16 bytes land in 1 KB in
// lane order), D / 8 pieces, W waves; the swizzle is applied to the source column.
// In asm: for the builtin the compiler waits for every load under way before it reads any LDS of the same array,
// which would make the prefetch of the next tile a wait for it.  No register is written; landed() and a
// barrier stand between these loads and the reads of their tile.
template <int D, int W>
struct Loader {
  static constexpr int P = D / (8 * W), RP = 512 / D;  // pieces per wave, rows per piece
  static constexpr int KINDS = RP % 8 ? 2 : 1;     // swz repeats every 8 rows: pieces of 4 rows come in two kinds
  static constexpr unsigned TILE = TK * D * 2;     // bytes
  unsigned off[KINDS];                              // this lane's source offset within a piece (bytes)
  unsigned to;                                      // this wave's first piece in buffer 0
  const char* base;                                 // row 0
  long step;                                        // bytes per row
  __device__ __forceinline__ void init(const unsigned short* b, long ls, const unsigned short* tile) {
    const int lane = threadIdx.x & 63;
    base = reinterpret_cast<const char*>(b);
    step = ls * 2;
    to = lds_at(tile) + (unsigned)(wave_id() * P * 1024);
#pragma unroll
    for (int k = 0; k < KINDS; ++k) {
      const int r = lane / (D / 8);
      off[k] = (unsigned)(r * (int)step) + (unsigned)(((lane % (D / 8)) ^ swz<D>(r + RP * k)) * 16);
    }
  }
  __device__ __forceinline__ void issue(int r0, int L, int buf) const {
    const unsigned t = to + (buf ? TILE : 0u);
    const int w0 = r0 + wave_id() * P * RP;  // this wave's first row
    const char* b = base + (long)w0 * step;
    if (r0 + TK <= L) {
#pragma unroll
      for (int u = 0; u < P; ++u) glds(b + (long)(u * RP) * step, off[u % KINDS], t + u * 1024);
    } else {  // rows behind the sequence: its last row again (their probabilities are zero)
      const int lane = threadIdx.x & 63;
      const char* b0 = base + (long)r0 * step;
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const int r = (w0 - r0) + u * RP + lane / (D / 8), c = (lane % (D / 8)) ^ swz<D>(r);
        glds(b0, (unsigned)min(r, L - 1 - r0) * (unsigned)step + c * 16, t + u * 1024);
      }
    }
  }
  static __device__ __forceinline__ void glds(const char* b, unsigned o, unsigned t) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(o), "s"(b), "s"(t) : "memory", "m0");
  }
};

// 64 floats x[r0 ..] of a row of L into LDS, by one wave
__device__ __forceinline__ void floats_to_lds(const float* x, int r0, int L, unsigned to) {
  const unsigned off = (unsigned)min((int)(threadIdx.x & 63), L - 1 - r0) * 4u;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(x + r0), "s"(to)
               : "memory", "m0");
}

// every load of this wave has arrived (in asm: the compiler does not know of the tile loads)
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// the same for the compiler's own loads, which it would otherwise wait for inside the loop
__device__ __forceinline__ void operands_here() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), the other counters unlimited
  __builtin_amdgcn_sched_barrier(0);
}

// Masked rows become zeros, so whatever they hold (infinities and NaN too) never meets a zero
// probability in a product.  Uniform over the workgroup; ends with a barrier.
template <int D, int W>
__device__ __forceinline__ void clear_rows(unsigned short* k, unsigned short* v, unsigned long long keep) {
#pragma unroll
  for (int u = 0; u < D / (8 * W); ++u) {
    const int c = threadIdx.x + 64 * W * u, r = c / (D / 8);
    if (!((keep >> r) & 1ull)) {
      *reinterpret_cast<u32x4*>(k + c * 8) = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4*>(v + c * 8) = u32x4{0, 0, 0, 0};
    }
  }
  __syncthreads();
}

// This lane's addresses within a tile.  A operand of a product: rows (lane & 31), columns 16 s + 8 (lane / 32).
// Transposed A operand: row = tile column (lane & 31) of a 32-column group; its 8 k-slots are the tile rows
// that registers 8 s .. 8 s + 7 of a 32 x 32 accumulator hold in this half-wave: 16 s + 4 h + {0..3}, +8.
// The swizzle touches other address bits than the row and the tile do, so a step in columns is an exclusive or
// with a constant: one register for each kind of address.
template <int D>
struct Frags {
  unsigned row, tr;  // bytes
  __device__ __forceinline__ void init() {
    const int lane = threadIdx.x & 63, h = lane >> 5, g = lane >> 4;
    row = (unsigned)((lane & 31) * D * 2 + (h ^ swz<D>(lane & 31)) * 16);
    const int r = 4 * (g >> 1) + ((lane & 15) >> 2), c = 16 * (g & 1) + 4 * (lane & 3);
    tr = (unsigned)(r * D * 2 + ((c >> 3) ^ swz<D>(r)) * 16 + (c & 7) * 2);
  }
  // rows r0 .. r0 + 31 (r0 a multiple of 32; swz repeats every 8 rows)
  __device__ __forceinline__ bf16x8 rows(const unsigned short* t, int r0, int s) const {
    return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(t) + (row ^ (32u * s)) + r0 * D * 2);
  }
  __device__ __forceinline__ bf16x8 trans(const unsigned short* t, int r0, int s, int e) const {
    const char* p = reinterpret_cast<const char*>(t) + (tr ^ (64u * e)) + (r0 + 16 * s) * D * 2;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 8 * D * 2));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};

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

__device__ __forceinline__ uint2 quad(const f32x16& x, int t, float scale) {
  return uint2{pack_bf16x2(x[4 * t] * scale, x[4 * t + 1] * scale), pack_bf16x2(x[4 * t + 2] * scale, x[4 * t + 3] * scale)};
}

__device__ __forceinline__ f32x16 splat16(float v) {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = v;
  return z;
}

// the same row's value in the other half-wave
__device__ __forceinline__ float other_half(float v, bool hi) {
  const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(hi ? r[0] : r[1]);
}

// bf16 quads t and t + 1 of this half-wave (columns 8 t + 4 h .., 8 (t + 1) + 4 h ..) -> the 8 columns 8 (t + h) ..: 16
// bytes to store at once, 32 to a row (by 8 and 16 bytes, forward and backward of 64 pages x 975 tokens x 12 heads took 455
// us instead of 414, of 4096 x 32 tokens 932 instead of 778)
__device__ __forceinline__ u32x4 eight(uint2 a, uint2 b) {
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false));
  const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false));
  return u32x4{x[0], y[0], x[1], y[1]};
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

// What the 32 queries w0 .. of a wave see of 32 keys j0 .. j0+31 with keep bits kw: scalars, a few compares per block
struct Sees {
  int none_lo, none_hi, full_lo, full_hi, sinks;
  __device__ __forceinline__ Sees(const Args& a, int w0) {
    none_lo = w0 - a.left - 31;
    none_hi = w0 < a.L ? w0 + 31 + a.right : -1;
    full_lo = w0 + 31 - a.left;
    full_hi = w0 + a.right - 31;
    sinks = a.sinks;
  }
  __device__ __forceinline__ int kind(int j0, unsigned kw) const {
    // outside / inside of an interval by the sign of the differences: a few scalar instructions, no branches
    const int out = (none_hi - j0) | ((j0 - none_lo) & (sinks - 1 - j0));
    const int over = (full_hi - j0) | ((j0 - full_lo) & (sinks - 32 - j0));
    if (out < 0 || kw == 0u) return EMPTY;
    return over >= 0 && kw == 0xFFFFFFFFu ? FULL : PARTIAL;
  }
};

// the keys of j0 .. j0+31 that query i sees, as bits
__device__ __forceinline__ unsigned seen_keys(const Args& a, int i, int j0, unsigned kw) {
  return kw & (bits_between(i - a.left - j0, i + a.right - j0) |
               (bits_between(0, a.sinks - 1 - j0) & bits_between(0, i + a.right - j0)));
}

// Workgroup -> (sequence and head, tile).  Workgroups go to the 8 XCDs in turn: the tiles of a head stay on one XCD,
// whose L2 then holds their keys, and heads are dealt to the XCDs one by one, so that pages of different
// lengths spread evenly (whole ranges of sequences per XCD measured 3 to 5 % slower on ragged pages).
struct Where {
  int nh, tile;
  __device__ __forceinline__ Where(int bid, int heads, int tiles) {
    const int even = heads / 8 * 8 * tiles;
    if (bid < even) {
      const int i = bid / 8;
      nh = i / tiles * 8 + bid % 8;
      tile = i % tiles;
    } else {
      const int r = heads % 8, i = bid - even;
      nh = heads - r + i % r;
      tile = i / r;
    }
  }
};

// Walks the key tiles that queries b0 .. b0 + RB - 1 see (the tiles of the sinks, then the window's):
// `each(tile K, tile V, first key, keep bits)`; `meanwhile()` while the first one is on its way.  While a tile is worked on, the next one is on its way to the
// other buffer.  The mask is read ahead for 128 tiles at once, as one word per tile in LDS: tiles without
// a key that counts cost nothing (a page's padding is such a run of tiles).  B = 1: there is one tile only.
template <int D, int W, int B, typename S, typename F>
__device__ __forceinline__ void walk_keys(const Args& a, int n, int kvh, int b0, unsigned short (&kt)[B][TK * D],
                                          unsigned short (&vt)[B][TK * D], unsigned long long (&words)[128], S meanwhile, F each) {
  const int lane = threadIdx.x & 63;
  const unsigned short* K = a.k.p + n * a.k.n + kvh * a.k.h;
  const unsigned short* V = a.v.p + n * a.v.n + kvh * a.v.h;
  Loader<D, W> lk, lv;
  lk.init(K, a.k.l, kt[0]);
  lv.init(V, a.v.l, vt[0]);
  const int lo = max(0, b0 - a.left) / TK, hi = min(a.L - 1, min(b0 + RB, a.L) - 1 + a.right) / TK;
  const int sink = min((a.sinks + TK - 1) / TK, lo), jump = lo - sink, tiles = sink + hi - lo + 1;
  unsigned long long some0 = 0ull, some1 = 0ull;  // tiles of this chunk of 128 that are still to come
  int first = 0, chunk = 0;                       // its first tile, the first tile behind it
  const unsigned long long tail = a.L % TK ? (1ull << (a.L % TK)) - 1ull : ~0ull;
  const int last = (a.L - 1) / TK;
  auto refill = [&]() {
    const int m = min(tiles - chunk, 128);
    first = chunk;
    if (a.mask) {
      __syncthreads();  // the last chunk's words have been read
      for (int t0 = 0; t0 < m; t0 += 4 * W) {
        int mk[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t = chunk + min(t0 + W * u + wave_id(), m - 1), r = (t < sink ? t : t + jump) * TK + lane;
          const long at = (long)n * a.mask_n + min(r, a.L - 1);
          mk[u] = a.mask_bytes == 1 ? (int)reinterpret_cast<const unsigned char*>(a.mask)[at]
                                    : reinterpret_cast<const int*>(a.mask)[at];
          if (r >= a.L) mk[u] = 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const unsigned long long w = __ballot(mk[u] != 0);
          const int t = t0 + W * u + wave_id();
          if (t < m && lane == 0) words[t] = w;
        }
      }
      __syncthreads();
      some0 = __ballot(lane < m && words[lane] != 0ull);
      some1 = __ballot(lane + 64 < m && words[lane + 64] != 0ull);
    } else {
      some0 = m >= 64 ? ~0ull : (1ull << m) - 1ull;
      some1 = m >= 128 ? ~0ull : m > 64 ? (1ull << (m - 64)) - 1ull : 0ull;
    }
    chunk += m;
  };
  // the next tile of the walk with a key that counts, or -1; its keep bits
  auto next = [&](unsigned long long& keep) -> int {
    while ((some0 | some1) == 0ull) {
      if (chunk >= tiles) return -1;
      refill();
    }
    int t = some0 ? __builtin_ctzll(some0) : 64 + __builtin_ctzll(some1);
    if (some0) some0 &= some0 - 1;
    else some1 &= some1 - 1;
    const int g = first + t, tile = g < sink ? g : g + jump;
    if (a.mask) {
      const unsigned long long w = words[t];
      keep = ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(w >> 32)) << 32) |
             (unsigned)__builtin_amdgcn_readfirstlane((unsigned)w);
    } else {
      keep = tile == last ? tail : ~0ull;
    }
    return tile;
  };
  auto read = [&](int tile, int buf) {
    lk.issue(tile * TK, a.L, buf % B);
    lv.issue(tile * TK, a.L, buf % B);
  };
  unsigned long long keep = 0ull, keep1;
  int t0, t1 = next(keep1), buf = 0;  // t0: the tile worked on; t1: the tile being read
  const bool any = t1 >= 0;
  if (any) read(t1, 0);
  meanwhile();
  operands_here();  // the first tile too
  if (!any) return;
  while (true) {
    __syncthreads();
    t0 = t1;
    keep = keep1;
    if (a.mask && keep != ~0ull) clear_rows<D, W>(kt[buf % B], vt[buf % B], keep);
    t1 = next(keep1);
    if (t1 >= 0) read(t1, buf ^ 1);
    each(kt[buf % B], vt[buf % B], t0 * TK, keep);
    if (t1 < 0) return;
    landed();
    buf ^= 1;
  }
}

// ------------------------------------------------------------------------------------ forward
// Workgroup = 128 queries of one head; a wave owns 32 of them (lane & 31), both half-waves hold the
// same queries and split the keys of each block.  Bound by instruction issue, vector and matrix about equally:
// 12 heads x 64, 32 ragged pages x 2000 tokens, window 256 + 256: 178 us (400 TFLOP/s of visible pairs, no
// rescaling of accumulators in nearly all blocks); all 2048 x 2048 pairs 500 - 590 us (820 - 700); 16 heads x 128,
// 4 x 4096 causal, window 1024: 197 (610).  Workgroups of 8 waves read the keys half as often and took 229
// against 187 us; 64 queries per wave 242 against 181 (registers).
template <int D, int W>
__global__ __launch_bounds__(64 * W, D <= 64 ? 4 : 2) void fwd_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) unsigned short kt[W / 2][TK * D];
  __shared__ __attribute__((aligned(1024))) unsigned short vt[W / 2][TK * D];
  __shared__ unsigned long long words[128];
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const Where wg(blockIdx.x, gridDim.x / a.tiles, a.tiles);
  const int hd = wg.nh % a.H, n = wg.nh / a.H;
  const int b0 = wg.tile * RB, w0 = b0 + wave_id() * 32, i = w0 + (lane & 31);
  const float sl = a.scale * LOG2E, slack = fminf(SLACK / sl, 1e30f);
  bf16x8 qf[D / 16];
  glob_frag<D>(a.q.p + n * a.q.n + (long)min(i, a.L - 1) * a.q.l + hd * a.q.h, i < a.L, qf);
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c] = splat16(0.f);
  float m = -INFINITY, ms = 0.f, l = 0.f;  // m: raw score, lags behind the maximum by at most SLACK; ms = -m sl
  Frags<D> fr;
  fr.init();
  const Sees sees(a, w0);
  walk_keys<D, W>(a, n, hd / a.G, b0, kt, vt, words, [] {}, [&](const unsigned short* k, const unsigned short* v, int j0, unsigned long long keep) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const unsigned kw = (unsigned)(keep >> (32 * c));
      const int kind = sees.kind(j0 + 32 * c, kw);
      if (kind == EMPTY) continue;
      f32x16 s = splat16(0.f);
#pragma unroll
      for (int t = 0; t < D / 16; ++t) s = MFMA32(fr.rows(k, 32 * c, t), qf[t], s);
      if (kind == PARTIAL) {
        const unsigned see = seen_keys(a, i, j0 + 32 * c, kw) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (see >> reg_bit(r)) & 1u ? s[r] : -INFINITY;
      }
      float bm = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[r]);
      bm = fmaxf(bm, other_half(bm, h));
      if (__ballot(bm > m + slack) != 0ull) {
        const float mn = fmaxf(m, bm);
        const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * sl);  // 0 at the first visible key
        l *= corr;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] *= corr;
        m = mn;
        ms = m == -INFINITY ? 0.f : -m * sl;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl, ms));
        l += s[r];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 pb = pack8(s, t);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = MFMA32(fr.trans(v, 32 * c, t, e), pb, o[e]);
      }
    }
  });
  l += other_half(l, h);
  if (i >= a.L) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  unsigned short* orow = a.o.p + n * a.o.n + (long)i * a.o.l + hd * a.o.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] *= inv;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      const uint2 w[2] = {quad(o[e], t, 1.f), quad(o[e], t + 1, 1.f)};
      *reinterpret_cast<u32x4*>(orow + e * 32 + 8 * (t + h)) = eight(w[0], w[1]);
      if (a.lse) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          unsigned rest = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            rest |= (unsigned)(rest_of(o[e][4 * (t + v) + u], ((u < 2 ? w[v].x : w[v].y) >> (16 * (u & 1))) & 0xffffu) & 0xff)
                    << (8 * u);
          *reinterpret_cast<unsigned*>(rest_at<D>(a, n, hd, i, 4 * e + t + v) + 4 * h) = rest;
        }
      }
    }
  if (a.lse && h == 0)
    a.lse[((long)n * a.H + hd) * a.L + i] = l == 0.f ? -INFINITY : -fmaf(m, sl, __log2f(l));
}

// ------------------------------------------------------------------------------------ backward: dq, D
// Same walk as the forward: dS^T in registers, dq^T += K^T dS^T.  D is the lane's own row sum of
// do * o and goes to memory for the other kernel; -D is the start value of the dP accumulators (from zero,
// subtracted later: 623 instead of 618 us, forward and backward of the forward's pages).  Those pages:
// 228 us; four waves per SIMD spill and cost 35 us.
template <int D, int W>
__global__ __launch_bounds__(64 * W, D <= 64 ? 3 : 2) void bwd_dq_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) unsigned short kt[W / 2][TK * D];
  __shared__ __attribute__((aligned(1024))) unsigned short vt[W / 2][TK * D];
  __shared__ unsigned long long words[128];
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const Where wg(blockIdx.x, gridDim.x / a.tiles, a.tiles);
  const int hd = wg.nh % a.H, n = wg.nh / a.H;
  const int b0 = wg.tile * RB, w0 = b0 + wave_id() * 32, i = w0 + (lane & 31), ic = min(i, a.L - 1);
  const float sl = a.scale * LOG2E;
  bf16x8 qf[D / 16], gf[D / 16];
  glob_frag<D>(a.q.p + n * a.q.n + (long)ic * a.q.l + hd * a.q.h, i < a.L, qf);
  glob_frag<D>(a.go.p + n * a.go.n + (long)ic * a.go.l + hd * a.go.h, i < a.L, gf);
  bf16x8 of[D / 16];
  glob_frag<D>(a.o.p + n * a.o.n + (long)ic * a.o.l + hd * a.o.h, i < a.L, of);
  uint2 rest[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) rest[s] = *reinterpret_cast<const uint2*>(rest_at<D>(a, n, hd, ic, 2 * s + h));
  const long row = ((long)n * a.H + hd) * a.L + ic;
  const float nlse = a.lse[row];
  f32x16 minus_d;
  auto row_sum = [&] {
    float dd = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        dd = fmaf(with_rest((unsigned short)of[s][e], (int)((e < 4 ? rest[s].x : rest[s].y) << (24 - 8 * (e & 3))) >> 24),
                  bf16_to_f32((unsigned short)gf[s][e]), dd);
    dd += other_half(dd, h);
    if (i < a.L && h == 0) a.dd[row] = -dd;
    minus_d = splat16(-dd);
  };
  f32x16 acc[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc[c] = splat16(0.f);
  Frags<D> fr;
  fr.init();
  const Sees sees(a, w0);
  walk_keys<D, W>(a, n, hd / a.G, b0, kt, vt, words, row_sum, [&](const unsigned short* k, const unsigned short* v, int j0, unsigned long long keep) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const unsigned kw = (unsigned)(keep >> (32 * c));
      const int kind = sees.kind(j0 + 32 * c, kw);
      if (kind == EMPTY) continue;
      f32x16 s = splat16(0.f), dp = minus_d;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        s = MFMA32(fr.rows(k, 32 * c, t), qf[t], s);
        dp = MFMA32(fr.rows(v, 32 * c, t), gf[t], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl, nlse)) * dp[r];
      if (kind == PARTIAL) {
        const unsigned see = seen_keys(a, i, j0 + 32 * c, kw) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (see >> reg_bit(r)) & 1u ? s[r] : 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 b = pack8(s, t);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = MFMA32(fr.trans(k, 32 * c, t, e), b, acc[e]);
      }
    }
  });
  if (i >= a.L) return;
  unsigned short* drow = a.dq.p + n * a.dq.n + (long)i * a.dq.l + hd * a.dq.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; t += 2)
      *reinterpret_cast<u32x4*>(drow + e * 32 + 8 * (t + h)) = eight(quad(acc[e], t, a.scale), quad(acc[e], t + 1, a.scale));
}

// ------------------------------------------------------------------------------------ backward: dk, dv
// Workgroup = 128 keys of one key/value head, a wave owns 32 of them; it walks the query tiles of
// every query head of the group: P and dS (queries x keys), dv^T += dO^T P, dk^T += Q^T dS.  The rows'
// -D are the start values of the dP accumulators, read from LDS into place.  The forward's pages: 269 us with
// the far queries; heads of 128: one wave per SIMD (321 registers), 414 us, and a tile's two blocks taken
// together, products under exponentials, need more than 512 (spills: 741 -> 976 us, forward and backward).
//
// The sinks are seen by every later query: walked by their own workgroup alone they would make it the last
// by far.  Their far queries (behind the window's tiles) are dealt to workgroups of FAR tiles each, whose
// waves share 32 keys and split the queries; partial sums in fp32, added up by sink_sum_kernel.  They
// are further workgroups of their head in the same launch, whose reads of Q and dO the others bring to the XCD's L2
// (a launch of their own: 47 + 174 us against 189 at 64 pages x 975 tokens x 12 heads, 4 sinks; in the dq kernel, which
// has the queries at hand, they cost as much as on their own).
template <int D>
struct KeyGrads {
  bf16x8 kf[D / 16], vf[D / 16];
  f32x16 dk[D / 32], dv[D / 32];
  // 32 queries (rows r0 .. of the tiles, ls / ds their -log-sum-exp and -D) against the wave's 32 keys
  __device__ __forceinline__ void block(const Frags<D>& fr, const unsigned short* qt, const unsigned short* gt, int r0,
                                        const float* ls, const float* ds, float sl, unsigned see, bool full) {
    const int h = (threadIdx.x & 63) >> 5;
    f32x16 p = splat16(0.f), dp;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(ds + 8 * t + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * t + e] = d4[e];
    }
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      p = MFMA32(fr.rows(qt, r0, t), kf[t], p);
      dp = MFMA32(fr.rows(gt, r0, t), vf[t], dp);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + 8 * t + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * t + e;
        p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], sl, l4[e]));
        dp[r] *= p[r];
      }
    }
    if (!full) {
      see >>= 4 * h;
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
        dv[e] = MFMA32(fr.trans(gt, r0, t, e), pb, dv[e]);
        dk[e] = MFMA32(fr.trans(qt, r0, t, e), sb, dk[e]);
      }
    }
  }
};

// Partial sums of the sinks, fp32: slots of [dk, dv][sink][D].  Lane's four values of accumulator quad t of column
// group e: d = 32 e + 8 t + 4 h ..
template <int D>
__device__ __forceinline__ float* part_at(const Args& a, long slot, int which, int key, int e, int t) {
  return a.part + ((slot * 2 + which) * a.sinks + key) * D + 32 * e + 8 * t + 4 * ((threadIdx.x & 63) >> 5);
}

// the wave's 32 keys w0 ..: whether this lane's counts, K and V in registers, sums cleared
template <int D>
__device__ __forceinline__ bool key_lane(const Args& a, int n, int kvh, int j, KeyGrads<D>& w) {
  const int jc = min(j, a.L - 1);
  bool ok = j < a.L;
  if (a.mask) {
    const long mi = (long)n * a.mask_n + jc;
    ok = ok && (a.mask_bytes == 1 ? (int)reinterpret_cast<const unsigned char*>(a.mask)[mi]
                                  : reinterpret_cast<const int*>(a.mask)[mi]) != 0;
  }
  glob_frag<D>(a.k.p + n * a.k.n + (long)jc * a.k.l + kvh * a.k.h, ok, w.kf);
  glob_frag<D>(a.v.p + n * a.v.n + (long)jc * a.v.l + kvh * a.v.h, ok, w.vf);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) w.dk[c] = w.dv[c] = splat16(0.f);
  return ok;
}

template <int D, int W, int B>
__global__ __launch_bounds__(64 * W, D <= 64 ? 3 : 1) void bwd_dkv_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) unsigned short tiles[2 * B][TK * D];  // Q .., dO ..
  __shared__ __attribute__((aligned(16))) float ls[B][TK], ds[B][TK];
  unsigned short(*const qt)[TK * D] = tiles, (*const gt)[TK * D] = tiles + B;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int Hkv = a.H / a.G;
  const Where wg(blockIdx.x, gridDim.x / (a.tiles + a.far_wgs), a.tiles + a.far_wgs);
  const int kvh = wg.nh % Hkv, n = wg.nh / Hkv;
  // far: (head of the group, chunk of query tiles, 32-key block of sinks)
  const bool far = W == 4 && wg.tile >= a.tiles;
  const int x = wg.tile - a.tiles, gc = far ? x / a.far_blocks : 0, g0 = far ? gc / a.far_chunks : 0;
  const int b0 = far ? 0 : wg.tile * RB, w0 = far ? x % a.far_blocks * 32 : b0 + wave_id() * 32, j = w0 + (lane & 31);
  const float sl = a.scale * LOG2E;
  const bool split = a.far_chunks != 0;
  KeyGrads<D> w;
  const bool ok = key_lane<D>(a, n, kvh, j, w);
  const unsigned long long okw = __ballot(ok);
  const bool all_ok = okw == ~0ull, any_ok = okw != 0ull;
  // queries that see a key of this workgroup: from b0 - right to the last key + left, or (sinks
  // that are not split off) to the end
  const int lo = far ? a.far_tile + gc % a.far_chunks * FAR : max(0, b0 - a.right) / TK;
  const int last = far ? min(a.L, (lo + FAR) * TK) - 1
                       : b0 < a.sinks && !split ? a.L - 1 : min(a.L - 1, min(b0 + RB, a.L) - 1 + a.left);
  const int per = last / TK - lo + 1, total = __syncthreads_or(any_ok) ? (far ? per : per * a.G) : 0;
  // the same three kinds as in the forward, seen from the wave's keys
  const int none_lo = w0 - a.right - 31, none_hi = !any_ok ? -1 : w0 < a.sinks ? a.L - 1 : min(a.L - 1, w0 + 31 + a.left);
  const int full_lo = w0 + 31 - a.right;
  const int full_hi = !all_ok ? -1 : w0 + 31 < a.sinks ? a.L - 32 : min(a.L - 32, w0 + a.left - 31);
  const int my_last = min(a.L - 1, j < a.sinks ? a.L - 1 : j + a.left);
  Frags<D> fr;
  fr.init();
  Loader<D, W> lq, lg;
  lq.init(a.q.p + n * a.q.n + (long)(kvh * a.G + g0) * a.q.h, a.q.l, qt[0]);
  lg.init(a.go.p + n * a.go.n + (long)(kvh * a.G + g0) * a.go.h, a.go.l, gt[0]);
  const float *rl = a.lse + ((long)n * a.H + kvh * a.G + g0) * a.L, *rd = a.dd + ((long)n * a.H + kvh * a.G + g0) * a.L;
  const unsigned ls_at = lds_at(ls[0]), ds_at = lds_at(ds[0]);
  int t1 = 0, i0t;  // the tile being read, within its head; the first query of the tile worked on
  auto read = [&](int buf) {
    const int r1 = (lo + t1) * TK;
    lq.issue(r1, a.L, buf % B);
    lg.issue(r1, a.L, buf % B);
    if (wave_id() == 0) floats_to_lds(rl, r1, a.L, ls_at + buf % B * TK * 4);
    if (wave_id() == 1) floats_to_lds(rd, r1, a.L, ds_at + buf % B * TK * 4);
  };
  if (total) read(0);
  operands_here();  // the first tile too
  for (int it = 0, buf = 0; it < total; ++it, buf ^= 1) {
    __syncthreads();
    i0t = (lo + t1) * TK;
    if (++t1 == per) {  // the group's next head
      t1 = 0;
      lq.base += a.q.h * 2;
      lg.base += a.go.h * 2;
      rl += a.L;
      rd += a.L;
    }
    if (it + 1 < total) read(buf ^ 1);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i0 = i0t + 32 * c;
      if (i0 < none_lo || i0 > none_hi || (far && 2 * (it & 1) + c != wave_id())) continue;
      const bool full = i0 >= full_lo && i0 <= full_hi;
      unsigned see = 0u;
      if (!full) see = ok ? bits_between(j - a.right - i0, my_last - i0) : 0u;
      w.block(fr, qt[buf % B], gt[buf % B], 32 * c, &ls[buf % B][32 * c], &ds[buf % B][32 * c], sl, see, full);
    }
    landed();
  }
  if (W == 4 && far) {  // the four waves' sums, added in wave order; wave wv finishes accumulator quad wv
    const int wv = wave_id();
    const long slot = a.far_main + ((long)n * a.H + kvh * a.G + g0) * a.far_chunks + gc % a.far_chunks;
    float* red = reinterpret_cast<float*>(&tiles[0][0]);  // 4 x 1024 floats
    static_assert(W < 4 || sizeof(tiles) >= 4 * 1024 * sizeof(float), "the waves' sums fit the tiles' place");
    auto finish = [&](const f32x16& x, int which, int e) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 16; ++r) red[wv * 1024 + r * 64 + lane] = x[r];
      __syncthreads();
      f32x4 y;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        y[q] = red[(4 * wv + q) * 64 + lane];
#pragma unroll
        for (int v = 1; v < 4; ++v) y[q] += red[v * 1024 + (4 * wv + q) * 64 + lane];
      }
      if (j < a.sinks) *reinterpret_cast<f32x4*>(part_at<D>(a, slot, which, j, e, wv)) = y;
    };
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      finish(w.dk[e], 0, e);
      finish(w.dv[e], 1, e);
    }
    return;
  }
  if (split && j < a.sinks) {  // the sinks' near part: added to the far ones
#pragma unroll
    for (int e = 0; e < D / 32; ++e)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 x, y;
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = w.dk[e][4 * t + q], y[q] = w.dv[e][4 * t + q];
        *reinterpret_cast<f32x4*>(part_at<D>(a, (long)n * Hkv + kvh, 0, j, e, t)) = x;
        *reinterpret_cast<f32x4*>(part_at<D>(a, (long)n * Hkv + kvh, 1, j, e, t)) = y;
      }
  }
  if (j >= a.L || (split && j < a.sinks)) return;
  unsigned short* kr = a.dk.p + n * a.dk.n + (long)j * a.dk.l + kvh * a.dk.h;
  unsigned short* vr = a.dv.p + n * a.dv.n + (long)j * a.dv.l + kvh * a.dv.h;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      *reinterpret_cast<u32x4*>(kr + e * 32 + 8 * (t + h)) = eight(quad(w.dk[e], t, a.scale), quad(w.dk[e], t + 1, a.scale));
      *reinterpret_cast<u32x4*>(vr + e * 32 + 8 * (t + h)) = eight(quad(w.dv[e], t, 1.f), quad(w.dv[e], t + 1, 1.f));
    }
}

// dk, dv of the sinks: near part + the group's heads' chunks, in that order.  Thread = element of a slot
// (2 x sinks x D), grid.y = sequence and key/value head.
__global__ __launch_bounds__(64) void sink_sum_kernel(Args a, int D) {
  const int Hkv = a.H / a.G, kvh = blockIdx.y % Hkv, n = blockIdx.y / Hkv;
  const int x = blockIdx.x * 64 + threadIdx.x, half = a.sinks * D;
  if (x >= 2 * half) return;
  const long set = 2L * half;
  float y = a.part[((long)n * Hkv + kvh) * set + x];
  for (int g = 0; g < a.G; ++g) {
    const float* far = a.part + (a.far_main + ((long)n * a.H + kvh * a.G + g) * a.far_chunks) * set + x;
#pragma unroll 8
    for (int c = 0; c < a.far_chunks; ++c) y += far[c * set];
  }
  const int which = x >= half, i = which ? x - half : x, j = i / D, d = i - j * D;
  const View& o = which ? a.dv : a.dk;
  o.p[n * o.n + (long)j * o.l + kvh * o.h + d] = f32_to_bf16(which ? y : y * a.scale);
}

#undef MFMA32

// operand i of a call: pointer and its three element strides st[3 i ..]
__host__ inline View view(const void* p, const long* st, int i) {
  return View{(unsigned short*)const_cast<void*>(p), st[3 * i], st[3 * i + 1], st[3 * i + 2]};
}

// A launch holds fewer than 2^32 threads along an axis
__host__ inline bool grid_holds(long workgroups, long L) { return workgroups * (L <= SHORT ? 128 : 256) < (1L << 32); }

// sizes that the kernels' 32-bit row arithmetic and their 1-D grids hold
__host__ inline int check_sizes(long N, long L, long H, long G, int d, float scale) {
  if (N <= 0 || L <= 0 || H <= 0 || G <= 0 || H % G) return -1;
  if (d != 32 && d != 64 && d != 128) return -2;
  if (L > (1L << 29) || !(scale > 0.f)) return -3;
  return grid_holds((L + RB - 1) / RB * H * N, L) ? 0 : -4;
}

// A row's offset within a tile of 64 is 32 bits of bytes: strides of the rows that tiles are read from (the l-th of the
// three of operand i)
__host__ inline bool tiles_hold(const long* st, int i) { return st[3 * i + 1] < (1L << 25); }

// The far part of the sinks is split off where they all lie in the first workgroup of keys and it is long
// enough to matter (8 tiles; forward and backward of 64 pages x 12 heads x 64, window 128 + 128, one sink, split / not:
// 5 tiles behind the window 356 / 352 us, 9 tiles 484 / 484, 15 tiles 682 / 715; 2 pages of 4096: 117 / 200).  More
// sinks than that fill several workgroups with long walks, which balance among themselves.
struct FarPlan {
  int wgs, chunks, blocks, tile;
  long near_slots, floats;
};
__host__ inline FarPlan far_plan(long N, long L, long H, long G, int d, int left, int sinks) {
  FarPlan f{};
  const long l = left < L ? left : L, tiles = (L + TK - 1) / TK;
  const long first = (RB - 1 + l < L - 1 ? RB - 1 + l : L - 1) / TK + 1;
  if (sinks <= 0 || sinks > RB || tiles - first < 8 || N * (H / G) > 65535) return f;
  f.tile = (int)first;
  f.chunks = (int)((tiles - first + FAR - 1) / FAR);
  f.blocks = (sinks + 31) / 32;
  const long wgs = G * f.blocks * f.chunks;
  if (!grid_holds((wgs + (L + RB - 1) / RB) * (H / G) * N, L)) return FarPlan{};
  f.wgs = (int)wgs;
  f.near_slots = N * (H / G);
  f.floats = (f.near_slots + N * H * f.chunks) * 2 * d * sinks;
  return f;
}

}  // namespace wattn
}  // namespace pv

using namespace pv;
using namespace pv::wattn;

namespace {
Args common(const void* q, const void* k, const void* v, const void* o, const long* st, const void* mask, long mask_n,
            int mask_bytes, float* lse, void* rest, int L, int H, int G, int left, int right, int sinks, float scale) {
  Args a{};
  a.q = view(q, st, 0);
  a.k = view(k, st, 1);
  a.v = view(v, st, 2);
  a.o = view(o, st, 3);
  a.mask = mask;
  a.mask_n = mask_n;
  a.mask_bytes = mask_bytes;
  a.lse = lse;
  a.rest = static_cast<unsigned char*>(rest);
  a.L = L, a.H = H, a.G = G;
  a.left = min(left, L), a.right = min(right, L), a.sinks = min(sinks, L);
  a.scale = scale;
  a.tiles = (L + RB - 1) / RB;
  return a;
}
}  // namespace

// q, o (N, L, H, d), k, v (N, L, H / G, d) bf16; st: element strides {n, l, h} of q, k, v, o
// (multiples of 8, 16-byte aligned pointers); left, right >= L: unbounded.  lse (N, H, L) fp32 and
// rest (N * H * ceil(L / 32) * 32 * d bytes) for the backward pass, or both null.
PV_API int pv_wattn_fwd(const void* q, const void* k, const void* v, void* o, const long* st, const void* mask,
                        long mask_n, int mask_bytes, float* lse, void* rest, int N, int L, int H, int G, int d,
                        int left, int right, int sinks, float scale, void* stream) {
  if (const int rc = check_sizes(N, L, H, G, d, scale)) return rc;
  if (!lse != !rest) return -5;
  if (!tiles_hold(st, 1) || !tiles_hold(st, 2)) return -6;
  const Args a = common(q, k, v, o, st, mask, mask_n, mask_bytes, lse, rest, L, H, G, left, right, sinks, scale);
  const dim3 grid((unsigned)((long)a.tiles * H * N));
  hipStream_t s = (hipStream_t)stream;
#define PV_WFWD(DV)                                                                                   \
  do {                                                                                                \
    if (L <= SHORT) hipLaunchKernelGGL((fwd_kernel<DV, 2>), grid, dim3(128), 0, s, a);                \
    else hipLaunchKernelGGL((fwd_kernel<DV, 4>), grid, dim3(256), 0, s, a);                           \
  } while (0)
  if (d == 32) PV_WFWD(32);
  else if (d == 64) PV_WFWD(64);
  else PV_WFWD(128);
#undef PV_WFWD
  PV_LAUNCH_CHECK();
  return 0;
}

// floats of workspace that pv_wattn_bwd needs besides dd
PV_API long pv_wattn_bwd_ws(int N, int L, int H, int G, int d, int left, int sinks) {
  return N > 0 && L > 0 && H > 0 && G > 0 ? far_plan(N, L, H, G, d, left, min(sinks, L)).floats : 0;
}

// st: strides of q, k, v, o, go, dq, dk, dv.  dd (N, H, L) and ws fp32 workspace; dq (N, L, H, d), dk, dv
// (N, L, H / G, d) bf16, every element written.
PV_API int pv_wattn_bwd(const void* q, const void* k, const void* v, const void* o, const void* go, void* dq, void* dk,
                        void* dv, const long* st, const void* mask, long mask_n, int mask_bytes, float* lse,
                        const void* rest, float* dd, float* ws, long ws_floats, int N, int L, int H, int G, int d, int left, int right, int sinks,
                        float scale, void* stream) {
  if (const int rc = check_sizes(N, L, H, G, d, scale)) return rc;
  for (const int i : {0, 1, 2, 4})  // q, k, v, go
    if (!tiles_hold(st, i)) return -6;
  Args a = common(q, k, v, o, st, mask, mask_n, mask_bytes, lse, const_cast<void*>(rest), L, H, G, left, right, sinks,
                  scale);
  a.go = view(go, st, 4);
  a.dq = view(dq, st, 5);
  a.dk = view(dk, st, 6);
  a.dv = view(dv, st, 7);
  a.dd = dd;
  const FarPlan f = far_plan(N, L, H, G, d, a.left, a.sinks);
  if (f.floats > 0 && (!ws || ws_floats < f.floats)) return -5;
  a.part = ws;
  a.far_chunks = f.chunks;
  a.far_blocks = f.blocks;
  a.far_tile = f.tile;
  a.far_main = f.near_slots;
  a.far_wgs = f.wgs;
  const dim3 gq((unsigned)((long)a.tiles * H * N)), gk((unsigned)((long)(a.tiles + f.wgs) * (H / G) * N));
  hipStream_t s = (hipStream_t)stream;
#define PV_WBWD(DV)                                                                                   \
  do {                                                                                                \
    if (L <= SHORT) hipLaunchKernelGGL((bwd_dq_kernel<DV, 2>), gq, dim3(128), 0, s, a);               \
    else hipLaunchKernelGGL((bwd_dq_kernel<DV, 4>), gq, dim3(256), 0, s, a);                          \
    PV_LAUNCH_CHECK();                                                                                \
    if (L <= SHORT && G == 1) hipLaunchKernelGGL((bwd_dkv_kernel<DV, 2, 1>), gk, dim3(128), 0, s, a); \
    else if (L <= SHORT) hipLaunchKernelGGL((bwd_dkv_kernel<DV, 2, 2>), gk, dim3(128), 0, s, a);      \
    else hipLaunchKernelGGL((bwd_dkv_kernel<DV, 4, 2>), gk, dim3(256), 0, s, a);                      \
    PV_LAUNCH_CHECK();                                                                                \
  } while (0)
  if (d == 32) PV_WBWD(32);
  else if (d == 64) PV_WBWD(64);
  else PV_WBWD(128);
#undef PV_WBWD
  if (f.wgs) {
    hipLaunchKernelGGL(sink_sum_kernel, dim3((2 * a.sinks * d + 63) / 64, (unsigned)(N * (H / G))), dim3(64), 0, s, a, d);
    PV_LAUNCH_CHECK();
  }
  return 0;
}
