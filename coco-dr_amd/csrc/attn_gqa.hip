// Attention over packed sequences with grouped heads for gfx950: any length, causal or within a window, head sizes up to 128.
//
//   s_ij = scale q_i . k_j      lse_i = log sum_j exp(s_ij)      p_ij = exp(s_ij - lse_i)      o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i        dp_ij = do_i . v_j               ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij do_i
//
// j runs over the keys that query i sees: those of its own sequence inside [i - left, i + right] whose mask entry is not zero;
// dk and dv also sum over the query heads of the key head's group.  A row that sees nothing has o = 0, lse = -inf and no gradients.
//
// The scores are formed transposed where a lane holds a query (S^T = K Q^T: softmax statistics are lane-local plus one exchange with
// lane ^ 32) and straight where it holds a key (dK, dV); in both the fp32 accumulators, rounded to bf16, are the next product's B
// operand as they stand, and that product's A operand is read from LDS with the transposing read in the same row order.
// bf16 is what the matrix pipe takes: P and dS are rounded to it (half a step, at most 2^-8 of each element); every sum is fp32.
#include <limits.h>
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "common.h"
#include "prof.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;  // where a running maximum starts: finite, so that a row without any key gives exp2(-inf - kLow) = 0 and no NaN
// A running maximum that is outgrown by less than 2^kGrow is left as it is: terms of up to 2^kGrow are as exact in fp32 and bf16 as those below 1, and
// the accumulators, at most 2^kGrow times a sum of |v|, stay finite.
constexpr float kGrow = 20.0f;
constexpr int kFar = 1 << 30;   // an unlimited window; i + kFar stays inside an int for every row index < 2^30
constexpr int BK = 64;          // rows of a staged tile

typedef cocodr_attn_gqa_args Args;

// ------------------------------------------------------------------------------------------------ tiles in LDS
// [rows][DP] bf16, DP = 64 or 128 (the head size rounded up; columns behind it are zeros).  The 16-byte chunks of a row are permuted
// so that both reads are free of bank conflicts: ds_read_b128 of 16 consecutive rows at one chunk, and the transposing read of 4
// consecutive rows x 4 chunks.
template <int DP> __device__ __forceinline__ int swz(int row) {
  if constexpr (DP == 64) return swz64(row);
  else return ((row & 3) << 2) | ((row >> 2) & 3);
}
template <int DP> __device__ __forceinline__ int tile_off(int row, int ch) { return row * (DP * 2) + ((ch ^ swz<DP>(row)) << 4); }

// operand fragment of rows r0 + (lane & 31), contraction columns 16 s + 8 (lane >> 5) .. + 7
template <int DP> __device__ __forceinline__ bf16x8 frag_rows(const char* t, int r0, int s, int lane) {
  return lds_read_b128(t, tile_off<DP>(r0 + (lane & 31), 2 * s + (lane >> 5)));
}
// operand fragment of the transposed tile: output row = column 32 dt + (lane & 31), contraction = tile rows rb + 4 (lane >> 5) + {0..3}
// and + 8: the rows that accumulator registers 8 j .. 8 j + 7 of a 32 x 32 product hold (rb = 16 j)
template <int DP> __device__ __forceinline__ bf16x8 frag_cols(const char* t, int rb, int dt, int lane) {
  const int g = lane >> 4, c = lane & 15;
  const int col = dt * 32 + ((g & 1) << 4) + ((c & 3) << 2);
  const int row = rb + ((g >> 1) << 2) + (c >> 2);
  const int within = (col & 7) << 1;
  return join_tr(lds_read_tr16(t, tile_off<DP>(row, col >> 3) + within), lds_read_tr16(t, tile_off<DP>(row + 8, col >> 3) + within));
}

// 16 (4) bytes a lane from a buffer into LDS, lane-linear from `dst`.  As an asm statement, because hipcc orders every later LDS read behind the
// builtin's vmcnt(0) - a tile on its way would be waited for in the middle of the one that is worked on.  The kernels wait themselves (dma_wait)
// before the barrier that hands a tile over.
typedef __attribute__((ext_vector_type(4))) uint32_t rsrc_t;
__device__ __forceinline__ rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  return rsrc_t{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, bytes, 0x00020000u};
}
// scalars that a vector instruction wrote may be read by a memory instruction five states later, and hipcc does not look into dma16
__device__ __forceinline__ void rsrc_settled(rsrc_t a) { asm volatile("s_nop 4" ::"s"(a)); }
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(LDS_PTR(const void))p; }
__device__ __forceinline__ void dma16(rsrc_t rs, uint32_t off, uint32_t more, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(rs), "s"(more), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void dma4(rsrc_t rs, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(rs), "s"(dst) : "memory", "m0");
}
// this wave's transfers are in LDS; with the barrier behind it, every wave's
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// BK rows of one head into a tile by LDS DMA: a wave's instruction (a piece) writes 1 KiB lane-linear, so the permutation goes into the source
// addresses.  Rows whose bit of `rows` is 0 (behind the sequence, masked out) and columns >= D are addressed behind the descriptor's
// end and arrive as zeros: whatever stands there in memory, NaN too, is not read.  The descriptor reaches over one tile only, so its
// 32-bit offsets do for any buffer.  Wave w has the pieces w, w + 4, ..: the permutation of its rows is the same in each, and a piece's
// offset differs from the first's by a scalar.
template <int DP> struct Stager {
  static constexpr int CH = DP / 8, RP = 64 / CH, PIECES = BK / RP / 4;  // chunks of a row, rows of a piece, pieces of a wave
  uint32_t ldb, span, first;  // bytes of a row, of a tile; this lane's offset in its wave's first piece
  int row;                    // the lane's row in it
  __device__ __forceinline__ Stager(long long ld, int D, int lane, int wid) {
    ldb = (uint32_t)ld * 2u;
    span = (uint32_t)(BK - 1) * ldb + (uint32_t)D * 2u;
    row = wid * RP + lane / CH;
    const int ch = (lane & (CH - 1)) ^ swz<DP>(row);
    first = ch * 8 < D ? (uint32_t)row * ldb + (uint32_t)ch * 16u : 0x80000000u;
  }
  __device__ __forceinline__ rsrc_t tile(const uint16_t* src) const { return rsrc_of(src, span); }
  // dst: the wave's first piece of the tile in LDS
  __device__ __forceinline__ void piece(int i, rsrc_t rs, uint32_t dst, uint64_t rows) const {
    uint32_t off = first;
    if (rows != ~0ull) off = (rows >> (row + i * 4 * RP)) & 1 ? first : 0x80000000u;
    dma16(rs, off, (uint32_t)(i * 4 * RP) * ldb, dst + i * 4096);
  }
  __device__ __forceinline__ void all(const uint16_t* src, uint32_t dst, uint64_t rows) const {
    const rsrc_t rs = tile(src);
    rsrc_settled(rs);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) piece(i, rs, dst, rows);
  }
};
// one row's operand fragments straight from memory (the operand that a wave keeps): zeros where `ok` is false and behind column D
template <int DP> __device__ __forceinline__ void load_frags(bf16x8 (&f)[DP / 16], const uint16_t* row, int D, bool ok, int half) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int col = (2 * s + half) * 8;
    f[s] = as_bf16x8(ok && col < D ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0u, 0u, 0u, 0u));
  }
}

// The loads that filled these have landed.  Without it hipcc waits for them where they are first used, inside the loop, with a vmcnt(0) that every turn
// of the loop then spends on the tile that was just sent for.
template <int N> __device__ __forceinline__ void landed(bf16x8 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("s_waitcnt vmcnt(0)" : "+v"(f[i]));
}

__device__ __forceinline__ bf16x8 pack_acc(const float* p, int j) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = p[j * 8 + e];
  return as_bf16x8(pack8(t));
}

// The maximum of 2 x 16 accumulators.  fmaxf costs a quieting v_max of every operand first, so the three-operand form is written out.  Its statements
// read results of the matrix pipe without hipcc knowing the instruction: the ordinary fmaxf in front reads both accumulators' results, waits
// for them, and every statement depends on its value.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
__device__ __forceinline__ float max32(const f32x16 (&s)[2]) {
  const float first = fmaxf(s[0][0], s[1][0]);
  float m[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    m[u] = first;
#pragma unroll
    for (int r = 1 + (u & 1) * 8; r + 1 < (u & 1 ? 16 : 9); r += 2) m[u] = max3(m[u], s[u >> 1][r], s[u >> 1][r + 1]);
  }
  return max3(max3(m[0], m[1], m[2]), m[3], max3(m[0], s[0][15], s[1][15]));
}
__device__ __forceinline__ float max16(const f32x16& s) {
  const float first = fmaxf(s[0], s[1]);
  const float a = max3(first, s[2], s[3]), b = max3(first, s[4], s[5]), c = max3(first, s[6], s[7]), d = max3(first, s[8], s[9]);
  return max3(max3(a, s[10], s[11]), max3(b, s[12], s[13]), max3(max3(c, s[14], s[15]), d, d));
}
// the maximum with, and the sum with, the lane 32 further on, which holds the other half of the row
struct Pair { float a, b; };
__device__ __forceinline__ Pair both_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const uint32_t a = r[0], b = r[1];
  return {__uint_as_float(a), __uint_as_float(b)};
}
__device__ __forceinline__ float max_halves(float v) {
  const Pair p = both_halves(v);
  return max3(p.a, p.b, p.a);
}
__device__ __forceinline__ float sum_halves(float v) {
  const Pair p = both_halves(v);
  return p.a + p.b;
}

// transposed accumulators (lane: row lane & 31, registers: columns 32 dt + 8 rg + 4 half + e) -> bf16 rows
template <int DP> __device__ __forceinline__ void store_T(uint16_t* row, const f32x16 (&o)[DP / 32], float mul, int D, bool ok, int half) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      float t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = o[dt][rg * 4 + e] * mul;
      const int d = dt * 32 + 8 * rg + 4 * half;
      if (ok && d < D) *reinterpret_cast<uint2*>(row + d) = pack4(t);
    }
}

// ------------------------------------------------------------------------------------------------ which rows a workgroup has
// The tiles of TILE rows are numbered without a table: tile t of sequence b has the number off[b] / TILE + b + t.  Rounding down and
// the + b leave a sequence at least as many numbers as it has tiles, so numbers do not collide, and there are T / TILE + B of them.
// Number -> sequence is the last b with off[b] / TILE + b <= number: a search 64 wide, one step up to 64 sequences.
struct Tile {
  int n, first, row0;  // the sequence's rows (0: nothing to do), this tile's first row in it, the sequence's first row in the buffer
};
template <int TILE> __device__ __forceinline__ Tile find_tile(const int32_t* off, int B, int T, int num, int lane) {
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int at = lo + lane * step;
    bool below = false;
    if (lane * step < n) below = min(max(off[at], 0), T) / TILE + at <= num;
    const int c = __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(below)));
    if (c == 0) break;
    const int cut = (c - 1) * step;
    n = min(step, n - cut);
    lo += cut;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int a = min(max(off[lo], 0), T), e = min(max(off[lo + 1], a), T);
  const int t = num - (a / TILE + lo);
  Tile r;
  r.n = t >= 0 && t < (e - a + TILE - 1) / TILE ? e - a : 0;
  r.first = t * TILE;
  r.row0 = a;
  return r;
}
// rows of the buffer that belong to no sequence: before the first and behind the last one
struct Gaps {
  int head, tail0, count;
  __device__ Gaps(const int32_t* off, int B, int T) {
    head = min(max(off[0], 0), T);
    tail0 = min(max(off[B], head), T);
    count = head + (T - tail0);
  }
  __device__ int row(int i) const { return i < head ? i : tail0 + (i - head); }
};

// bit r of the result: lo <= r < hi
__device__ __forceinline__ uint32_t bits32(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? ~0u : (hi <= 0 ? 0u : (1u << hi) - 1u);
  const uint32_t below_lo = lo >= 32 ? ~0u : (lo <= 0 ? 0u : (1u << lo) - 1u);
  return below_hi & ~below_lo;
}
__device__ __forceinline__ uint64_t bits_below(int n) { return n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1ull); }

// which of the BK keys from k0 on exist and are not masked out.  The load is started (key_word_load) one tile before its ballot is taken.
__device__ __forceinline__ int key_word_load(const int32_t* mask, int row0, int n, int k0, int lane) {
  return mask && k0 + lane < n ? mask[row0 + k0 + lane] : 1;
}
__device__ __forceinline__ uint64_t key_word(const int32_t* mask, int loaded, int n, int k0) {
  const uint64_t w = bits_below(n - k0);
  return mask ? w & __ballot(loaded != 0) : w;
}

// ------------------------------------------------------------------------------------------------ forward
__device__ __forceinline__ void fill_gaps(const Args& a, uint16_t* ctx, float* lse, int tid) {
  const Gaps gap(a.seq_off, a.B, a.T);
  for (long long i = blockIdx.x; i < (long long)gap.count * a.heads; i += gridDim.x) {
    const int row = gap.row((int)(i / a.heads)), h = (int)(i % a.heads);
    if (tid * 4 < a.dim) *reinterpret_cast<uint2*>(ctx + row * a.o_row + h * a.o_head + tid * 4) = make_uint2(0u, 0u);
    if (tid == 0) lse[(size_t)h * a.T + row] = -INFINITY;
  }
}

// A workgroup has 128 query rows of one head, each of its four waves 32 of them; K and V pass through LDS in tiles of 64 keys, two
// tiles each, so that a tile is on its way while the one before is worked on.
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_gqa_fwd_kernel(const Args a, uint16_t* __restrict__ ctx, float* __restrict__ lse, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) fill_gaps(a, ctx, lse, tid);
  const int slots = gridDim.x / a.heads, G = a.heads / a.kv_heads;
  const int unit = blockIdx.x % a.heads, kvh = unit % a.kv_heads, h = kvh * G + unit / a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, slots - 1 - (int)(blockIdx.x / a.heads), lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int q0 = tile.first + wid * 32, qi = q0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(q0 + 31, n - 1);
  const int kbeg = max(tile.first - left, 0) & ~(BK - 1), kend = min(last + right + 1, n);
  const uint16_t* kb_ = a.k + (long long)tile.row0 * a.k_row + kvh * a.k_head;
  const uint16_t* vb_ = a.v + (long long)tile.row0 * a.v_row + kvh * a.v_head;
  const float sl2 = a.scale * kLog2e;

  bf16x8 qf[DP / 16];
  load_frags<DP>(qf, a.q + (long long)(tile.row0 + qi) * a.q_row + h * a.q_head, a.dim, qi < n, half);
  landed(qf);
  f32x16 o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = kLow, l = 0.f;

  constexpr int TB = BK * DP * 2;  // bytes of a tile
  const uint32_t lds0 = lds_addr(smem) + wid * 1024;  // (this wave's first piece)
  const Stager<DP> sk(a.k_row, a.dim, lane, wid), sv(a.v_row, a.dim, lane, wid);
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  if (kbeg < kend) {
    sk.all(kb_ + kbeg * a.k_row, lds0, word);
    sv.all(vb_ + kbeg * a.v_row, lds0 + TB, word);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
    const char* Kt = smem + buf * 2 * TB;
    const char* Vt = Kt + TB;
    dma_wait();
    __syncthreads();
    const uint64_t next = key_word(a.mask, loaded, n, k0 + BK);
    if (k0 + BK < kend) {
      const uint32_t to = lds0 + (buf ^ 1) * 2 * TB;
      sk.all(kb_ + (long long)(k0 + BK) * a.k_row, to, next);
      sv.all(vb_ + (long long)(k0 + BK) * a.v_row, to + TB, next);
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
    }
    const uint64_t now = word;
    word = next;
    if (q0 >= n || k0 > wlast + right || k0 + BK <= q0 - left || now == 0) continue;  // this wave's rows see nothing of the tile
    f32x16 s[2];
    bf16x8 f0[DP / 16], f1[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) f0[c] = frag_rows<DP>(Kt, 0, c, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      f1[c] = frag_rows<DP>(Kt, 32, c, lane);
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f0[c], qf[c], s[0], 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 vf[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) vf[dt] = frag_cols<DP>(Vt, 0, dt, lane);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f1[c], qf[c], s[1], 0, 0, 0);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (now != ~0ull || k0 < wlast - left || k0 + BK > q0 + right + 1) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int base = k0 + kb * 32;
        const uint32_t see = (bits32(qi - left - base, qi + right + 1 - base) & (uint32_t)(now >> (kb * 32))) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = (see >> (8 * (r >> 2) + (r & 3))) & 1 ? s[kb][r] : -INFINITY;
      }
    }
    const float top = max_halves(max32(s)) * sl2;
    if (__any(top > m + kGrow)) {
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
    }
    // P of a 16-key step is made while the products of the step before run; the step's rows of V are fetched one step ahead
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float p[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[t >> 1][(t & 1) * 8 + r], sl2, -m));
        l += p[r];
      }
      const bf16x8 pf = as_bf16x8(pack8(p));
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[dt], pf, o[dt], 0, 0, 0);
        if (t < 3) vf[dt] = frag_cols<DP>(Vt, (t + 1) * 16, dt, lane);
      }
    }
  }
  l = sum_halves(l);
  if (qi < n && lane < 32) lse[(size_t)h * a.T + tile.row0 + qi] = l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
  store_T<DP>(ctx + (long long)(tile.row0 + qi) * a.o_row + h * a.o_head, o, l > 0.f || l != l ? 1.0f / l : 0.f, a.dim, qi < n, half);
}

// The same for long sequences, 64 query rows a wave and one wave a SIMD: every fragment of K and V that is read from LDS serves two products
// instead of one.  With 32 rows a wave the fragments of a 128-wide head take 1128 clocks of the compute unit's LDS per tile, the products 1024 of the
// matrix pipe.  With one wave there is no other to fill its waits, so the work is laid out for overlap in one instruction stream, in steps of 32 keys:
//   the scores of step i (16 MFMAs)        beside   the first half of step i - 1's exponentials
//   that half's 8 MFMAs of P V             beside   the second half's exponentials
//   the second half's 8                    beside   the maximum of step i's scores
// K and V have three tiles each, as the last step of a tile still reads V behind the barrier that opens the next.
//
// The 128 accumulators of the output stay in AGPRs: their products are asm statements (hipcc would copy accumulators to VGPRs and back around every
// branch).  What reads or changes them comes behind s_nops (acc_scale, acc_done), as hipcc does not know that the matrix pipe wrote them.
// FRESH: the B operand was packed just before (a vector instruction's result may be read by the matrix pipe two states later).
template <bool FRESH> __device__ __forceinline__ void mfma_acc(f32x16& o, const bf16x8& x, const bf16x8& y) {
  if constexpr (FRESH) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(x), "v"(y));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(x), "v"(y));
}
#define ACC_MUL(i) "v_accvgpr_read_b32 %16, %" #i "\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %" #i ", %16\n\t"
__device__ __forceinline__ void acc_scale(f32x16& o, float f) {
  float e[16], t;
#pragma unroll
  for (int r = 0; r < 16; ++r) e[r] = o[r];
  asm volatile("s_nop 15\n\ts_nop 15\n\t" ACC_MUL(0) ACC_MUL(1) ACC_MUL(2) ACC_MUL(3) ACC_MUL(4) ACC_MUL(5) ACC_MUL(6) ACC_MUL(7) ACC_MUL(8) ACC_MUL(9)
                   ACC_MUL(10) ACC_MUL(11) ACC_MUL(12) ACC_MUL(13) ACC_MUL(14) ACC_MUL(15) "s_nop 4"
               : "+a"(e[0]), "+a"(e[1]), "+a"(e[2]), "+a"(e[3]), "+a"(e[4]), "+a"(e[5]), "+a"(e[6]), "+a"(e[7]), "+a"(e[8]), "+a"(e[9]), "+a"(e[10]),
                 "+a"(e[11]), "+a"(e[12]), "+a"(e[13]), "+a"(e[14]), "+a"(e[15]), "=&v"(t)
               : "v"(f));
#pragma unroll
  for (int r = 0; r < 16; ++r) o[r] = e[r];
}
#undef ACC_MUL
__device__ __forceinline__ void acc_done(f32x16& o) { asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o)); }
// scores: QA: that operand stays in AGPRs, too.  What reads the result comes behind other products or score_done
template <bool FIRST, bool QA> __device__ __forceinline__ void mfma_score(f32x16& s, const bf16x8& k, const bf16x8& q) {
  if constexpr (FIRST && QA) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "a"(q));
  else if constexpr (FIRST) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "v"(q));
  else if constexpr (QA) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "a"(q));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "v"(q));
}
__device__ __forceinline__ void score_done(f32x16 (&s)[2]) { asm volatile("s_nop 15\n\ts_nop 15" : "+v"(s[0]), "+v"(s[1])); }
// f(0), f(1), .. f(N - 1) with the index as a constant
template <int N, class F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}
#define SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)

// A wave that is alone issues an instruction every 5 to 6 clocks, so their number counts as much as their kind: the LDS addresses of the fragments
// live in registers and move by one addition a tile, and a tile whose rows are all there is sent for with three instructions a piece.
template <int DP> struct Frags {
  uint32_t rows[DP / 16], cols[DP / 16];  // of row fragments 0, 1, .. and of column fragments (dt, rows 0 / 8) of a tile
  __device__ __forceinline__ Frags(uint32_t tile_rows, uint32_t tile_cols, int lane) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      rows[i] = tile_rows + tile_off<DP>(lane & 31, 2 * i + (lane >> 5));
      const int col = (i >> 1) * 32 + ((g & 1) << 4) + ((c & 3) << 2), row = ((g >> 1) << 2) + (c >> 2) + (i & 1) * 8;
      cols[i] = tile_cols + tile_off<DP>(row, col >> 3) + ((col & 7) << 1);
    }
  }
  static __device__ __forceinline__ void move(uint32_t (&at)[DP / 16], uint32_t by) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      at[i] += by;
      asm volatile("" : "+v"(at[i]));  // (it stays a register: hipcc would add it up again at every use)
    }
  }
  template <int ROW> __device__ __forceinline__ bf16x8 row(int c) const { return *(const LDS_PTR(bf16x8))(rows[c] + ROW * DP * 2); }
  template <int ROW> __device__ __forceinline__ bf16x8 col(int dt) const {
    return join_tr(__builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(cols[2 * dt] + ROW * DP * 2)),
                   __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(cols[2 * dt + 1] + ROW * DP * 2)));
  }
};

template <int DP>
__global__ __launch_bounds__(256, 1) void attn_gqa_fwd2_kernel(const Args a, uint16_t* __restrict__ ctx, float* __restrict__ lse, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) fill_gaps(a, ctx, lse, tid);
  const int slots = gridDim.x / a.heads, G = a.heads / a.kv_heads;
  const int unit = blockIdx.x % a.heads, kvh = unit % a.kv_heads, h = kvh * G + unit / a.kv_heads;
  const Tile tile = find_tile<256>(a.seq_off, a.B, a.T, slots - 1 - (int)(blockIdx.x / a.heads), lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int q0 = tile.first + wid * 64, qi = q0 + (lane & 31);
  const int last = min(tile.first + 255, n - 1), wlast = min(q0 + 63, n - 1);
  const int kbeg = max(tile.first - left, 0) & ~(BK - 1), kend = min(last + right + 1, n);
  const int wbeg = max(q0 - left, 0), wend = q0 < n ? min(wlast + right + 1, n) : 0;  // the keys that this wave's rows see
  const int allbeg = wlast - left, allend = q0 + right + 1;                           // ... that all of them see
  const uint16_t* ks = a.k + (long long)(tile.row0 + kbeg) * a.k_row + kvh * a.k_head;  // the tile that is sent for next
  const uint16_t* vs = a.v + (long long)(tile.row0 + kbeg) * a.v_row + kvh * a.v_head;
  const float sl2 = a.scale * kLog2e;

  constexpr int TB = BK * DP * 2, PIECES = Stager<DP>::PIECES, NC = DP / 16, ND = DP / 32;
  const uint32_t lds0 = lds_addr(smem), mine = lds0 + wid * 1024;  // (this wave's first piece)
  const Stager<DP> sk(a.k_row, a.dim, lane, wid), sv(a.v_row, a.dim, lane, wid);
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  sk.all(ks, mine, word);
  sv.all(vs, mine + TB, word);

  bf16x8 qf[2][NC];
#pragma unroll
  for (int b = 0; b < 2; ++b) load_frags<DP>(qf[b], a.q + (long long)(tile.row0 + qi + 32 * b) * a.q_row + h * a.q_head, a.dim, qi + 32 * b < n, half);
  f32x16 o[2][ND];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][dt][r] = 0.f;
  float m[2] = {kLow, kLow}, l[2] = {0.f, 0.f};
  f32x16 sA[2], sB[2];  // the scores of a tile's first and second 32 keys
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) sA[b][r] = sB[b][r] = -INFINITY;
  Frags<DP> f(lds0, lds0 + TB, lane);
  landed(qf[0]);
  landed(qf[1]);
#pragma unroll
  for (int c = 0; c < NC; ++c) asm volatile("s_nop 1" : "+a"(qf[1][c]));  // (from here on in AGPRs)

  // Registers 8 j + 2 i and the next of block b's scores: their exponentials, and from these the sum and the packed pair - a slot apart, as a
  // result is 8 clocks away
  float ex[2], ey[2];
  auto expo = [&](const f32x16 (&s)[2], int r, int b, const float (&m)[2]) {
    ex[b] = __builtin_amdgcn_exp2f(fmaf(s[b][r], sl2, -m[b]));
    ey[b] = __builtin_amdgcn_exp2f(fmaf(s[b][r + 1], sl2, -m[b]));
  };
  auto pack = [&](uint32_t (&w)[2], int b) {
    l[b] += ex[b];
    w[b] = pack2bf(ex[b], ey[b]);
    l[b] += ey[b];
  };
  auto operand = [](const uint32_t (&w)[4][2], int b) { return as_bf16x8(make_uint4(w[0][b], w[1][b], w[2][b], w[3][b])); };
  // One step of 32 keys from k0 (rows ROW .. of the tile): its scores into s where the wave's rows see some of them (now), and the probabilities and
  // products of the step before (scores sp, rows 32 - ROW .. of its tile; in front of a wave's first step an empty one, with scores of -inf).  send(i)
  // sends for piece i of the next tile.
  // Each product is followed by what fits into its 32 clocks.
  auto step = [&](auto row_, int now, auto&& send, int k0, uint32_t word, f32x16 (&s)[2], const f32x16 (&sp)[2]) {
    constexpr int ROW = decltype(row_)::value, RP = 32 - ROW;
    bf16x8 vf[ND];
    uint32_t w[4][2], x[4][2];
    if (now) {
      bf16x8 kf[NC];
      SCHED_FENCE();
#pragma unroll
      for (int c = 0; c < NC / 2; ++c) kf[c] = f.template row<ROW>(c);
      expo(sp, 0, 0, m);
      expo(sp, 0, 1, m);
      pack(w[0], 0);
      pack(w[0], 1);
      SCHED_FENCE();
#pragma unroll
      for (int t = 0; t < 2 * NC; ++t) {
        const int c = t >> 1, b = t & 1;
        if (t < 2) b ? mfma_score<true, true>(s[1], kf[0], qf[1][0]) : mfma_score<true, false>(s[0], kf[0], qf[0][0]);
        else b ? mfma_score<false, true>(s[1], kf[c], qf[1][c]) : mfma_score<false, false>(s[0], kf[c], qf[0][c]);
        if (b == 0) {
          if (c + NC / 2 < NC) kf[c + NC / 2] = f.template row<ROW>(c + NC / 2);
          else if (c - NC / 2 < ND) vf[c - NC / 2] = f.template col<RP>(c - NC / 2);
        } else if (c % (NC / PIECES) == NC / PIECES - 1) send(c / (NC / PIECES));
        // six pairs of registers are left: in every other slot of a half's exponentials, in the one behind it the sum
        constexpr int PER = 2 * NC / 4;  // slots for one pair's two blocks
        if (t / PER < 3) {
          const int i = t / PER + 1, u = t % PER;
          if (u == 0) expo(sp, 2 * i, 0, m);
          if (u == PER / 4) pack(w[i], 0);
          if (u == PER / 2) expo(sp, 2 * i, 1, m);
          if (u == PER / 2 + PER / 4) pack(w[i], 1);
        }
        SCHED_FENCE();
      }
      if (word != ~0u || k0 < allbeg || k0 + 32 > allend) {
        score_done(s);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int at = qi + 32 * b - k0;
          const uint32_t see = (bits32(at - left, at + right + 1) & word) >> (4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = (see >> (8 * (r >> 2) + (r & 3))) & 1 ? s[b][r] : -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) send(i);
      float mm[2] = {m[0], m[1]};
      asm volatile("" : "+v"(mm[0]), "+v"(mm[1]));  // (or hipcc makes the two branches' probabilities one, in front of both, beside nothing)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        expo(sp, 2 * i, 0, mm);
        expo(sp, 2 * i, 1, mm);
        pack(w[i], 0);
        pack(w[i], 1);
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) vf[dt] = f.template col<RP>(dt);
    }
    SCHED_FENCE();
    float top[2];
    {
      bf16x8 vg[ND];
      constexpr int UNITS = 8 / (2 * ND);  // (pair, block)s of the second half for each product of the first
      each<2 * ND>([&](auto t_) {
        constexpr int t = decltype(t_)::value, dt = t >> 1, b = t & 1;
        mfma_acc<(t < 2)>(o[b][dt], vf[dt], operand(w, b));
        if (b == 0) vg[dt] = f.template col<RP + 16>(dt);
#pragma unroll
        for (int u = t * UNITS; u < (t + 1) * UNITS; ++u) {
          if (u > 0) pack(x[(u - 1) >> 1], (u - 1) & 1);
          expo(sp, 8 + 2 * (u >> 1), u & 1, m);
        }
        SCHED_FENCE();
      });
      pack(x[3], 1);
      float t0[2] = {0.f, 0.f}, t1[2] = {0.f, 0.f};
      each<2 * ND>([&](auto t_) {
        constexpr int t = decltype(t_)::value, dt = t >> 1, b = t & 1;
        mfma_acc<(t < 2)>(o[b][dt], vg[dt], operand(x, b));
        // the maximum of s[b] in two chains, four registers of each a slot
#pragma unroll
        for (int u = t * 8 / (2 * ND); u < (t + 1) * 8 / (2 * ND); ++u) {
          const int y = u >> 1, q = u & 1;  // registers 4 y .. of block q
          if (y == 0) t0[q] = t1[q] = fmaxf(s[q][0], s[q][1]);
          t0[q] = max3(t0[q], s[q][4 * y], s[q][4 * y + 1]);
          t1[q] = max3(t1[q], s[q][4 * y + 2], s[q][4 * y + 3]);
        }
        SCHED_FENCE();
      });
      top[0] = max3(t0[0], t1[0], t1[0]);
      top[1] = max3(t0[1], t1[1], t1[1]);
    }
    if (now) {
#pragma unroll
      for (int b = 0; b < 2; ++b) top[b] = max_halves(top[b]) * sl2;
      if (__any(top[0] > m[0] + kGrow || top[1] > m[1] + kGrow)) {
        const bool old = __any((top[0] > m[0] + kGrow && m[0] > kLow) || (top[1] > m[1] + kGrow && m[1] > kLow));
        float f[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float up = top[b] > m[b] + kGrow ? top[b] : m[b];
          f[b] = __builtin_amdgcn_exp2f(m[b] - up);
          m[b] = up;
          l[b] *= f[b];
        }
        if (old)  // (rows whose first maximum this is have their accumulators at zero, the others' factors are 1)
          each<2 * ND>([&](auto i) { acc_scale(o[decltype(i)::value / ND][decltype(i)::value % ND], f[decltype(i)::value / ND]); });
      }
    }
  };

  // pieces of a whole tile: offsets of the wave's second, third, .. from its first
  uint32_t ko[PIECES], vo[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    ko[i] = (uint32_t)(i * 4 * Stager<DP>::RP) * sk.ldb;
    vo[i] = (uint32_t)(i * 4 * Stager<DP>::RP) * sv.ldb;
  }
  int buf = 0;
  int open = 0;
  uint32_t shift = 0;  // from the tile before to this one
  for (int k0 = kbeg; k0 < kend; k0 += BK) {
    dma_wait();
    __syncthreads();
    const uint64_t now = word;
    word = key_word(a.mask, loaded, n, k0 + BK);
    const int ahead = buf == 2 ? 0 : buf + 1;
    const uint32_t to = mine + ahead * 2 * TB;
    ks += BK * a.k_row;
    vs += BK * a.v_row;
    const rsrc_t rk = sk.tile(ks), rv = sv.tile(vs);
    // The next tile's K is sent for during the first step, its V during the second (eight pieces at once would hold the wave for over 1000 clocks) -
    // if all its rows are there: else at once.
    const int whole = __builtin_amdgcn_readfirstlane(k0 + BK < kend && word == ~0ull);
    if (k0 + BK < kend) {
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
      rsrc_settled(rk);
      if (!whole) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          sk.piece(i, rk, to, word);
          sv.piece(i, rv, to + TB, word);
        }
      }
    }
    auto send_k = [&](int i) { if (whole) dma16(rk, sk.first, ko[i], to + i * 4096); };
    auto send_v = [&](int i) { if (whole) dma16(rv, sv.first, vo[i], to + TB + i * 4096); };
    const int first = __builtin_amdgcn_readfirstlane(k0 < wend && k0 + 32 > wbeg), second = __builtin_amdgcn_readfirstlane(k0 + 32 < wend && k0 + 64 > wbeg);
    Frags<DP>::move(f.rows, shift);
    if (first || open) step(std::integral_constant<int, 0>{}, first, send_k, k0, (uint32_t)now, sA, sB);
    else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) send_k(i);
    }
    Frags<DP>::move(f.cols, shift);
    if (second || first) step(std::integral_constant<int, 32>{}, second, send_v, k0 + 32, (uint32_t)(now >> 32), sB, sA);
    else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) send_v(i);
    }
    open = second;
    shift = ahead == 0 ? -4 * TB : 2 * TB;
    buf = ahead;
  }
  if (open) {  // the last step's probabilities and products
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          expo(sB, j * 8 + 2 * i, b, m);
          pack(w[i], b);
        }
      each<2 * ND>([&](auto t_) {
        constexpr int t = decltype(t_)::value, dt = t >> 1, b = t & 1;
        mfma_acc<true>(o[b][dt], j == 0 ? f.template col<32>(dt) : f.template col<48>(dt), operand(w, b));
      });
    }
  }
  each<2 * ND>([&](auto i) { acc_done(o[decltype(i)::value / ND][decltype(i)::value % ND]); });
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int row = qi + 32 * b;
    const float t = sum_halves(l[b]);
    if (row < n && lane < 32) lse[(size_t)h * a.T + tile.row0 + row] = t > 0.f ? (m[b] + __log2f(t)) * kLn2 : (t == 0.f ? -INFINITY : t);
    store_T<DP>(ctx + (long long)(tile.row0 + row) * a.o_row + h * a.o_head, o[b], t > 0.f || t != t ? 1.0f / t : 0.f, a.dim, row < n, half);
  }
}

// ------------------------------------------------------------------------------------------------ backward
// dQ: 128 query rows of one head a workgroup, 32 a wave (lane = query), over tiles of 64 keys as in the forward.  A wave has its rows of dO in
// registers: with ctx beside them it also makes -delta and -lse (in log2 units) of its rows and leaves them, [heads][T] each, for the dK / dV kernel.
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_gqa_dq_kernel(const Args a, const uint16_t* __restrict__ ctx, const uint16_t* __restrict__ dctx,
                                                             const float* __restrict__ lse, float* __restrict__ ndelta, float* __restrict__ nlse,
                                                             uint16_t* __restrict__ dq, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) {
    const Gaps gap(a.seq_off, a.B, a.T);
    for (long long i = blockIdx.x; i < (long long)gap.count * a.heads; i += gridDim.x)
      if (tid * 4 < a.dim) *reinterpret_cast<uint2*>(dq + gap.row((int)(i / a.heads)) * a.dq_row + (int)(i % a.heads) * a.dq_head + tid * 4) = make_uint2(0u, 0u);
  }
  const int slots = gridDim.x / a.heads, G = a.heads / a.kv_heads;
  const int unit = blockIdx.x % a.heads, kvh = unit % a.kv_heads, h = kvh * G + unit / a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, slots - 1 - (int)(blockIdx.x / a.heads), lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int q0 = tile.first + wid * 32, qi = q0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(q0 + 31, n - 1);
  const int kbeg = max(tile.first - left, 0) & ~(BK - 1), kend = min(last + right + 1, n);
  const uint16_t* kb_ = a.k + (long long)tile.row0 * a.k_row + kvh * a.k_head;
  const uint16_t* vb_ = a.v + (long long)tile.row0 * a.v_row + kvh * a.v_head;
  const float sl2 = a.scale * kLog2e;

  bf16x8 qf[DP / 16], df[DP / 16];
  load_frags<DP>(qf, a.q + (long long)(tile.row0 + qi) * a.q_row + h * a.q_head, a.dim, qi < n, half);
  load_frags<DP>(df, dctx + (long long)(tile.row0 + qi) * a.do_row + h * a.do_head, a.dim, qi < n, half);
  const size_t at = (size_t)h * a.T + tile.row0 + qi;
  float nl = qi < n ? -lse[at] * kLog2e : 0.f;
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(nl));
  float nd = 0.f;
  {
    bf16x8 of[DP / 16];
    load_frags<DP>(of, ctx + (long long)(tile.row0 + qi) * a.o_row + h * a.o_head, a.dim, qi < n, half);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      float x[8], y[8];
      unpack8(__builtin_bit_cast(uint4, of[c]), x);
      unpack8(__builtin_bit_cast(uint4, df[c]), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) nd = fmaf(-x[e], y[e], nd);
    }
    nd = sum_halves(nd);
  }
  landed(qf);
  landed(df);
  if (qi < n && lane < 32) {
    ndelta[at] = nd;
    nlse[at] = nl;
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

  constexpr int TB = BK * DP * 2;
  const uint32_t lds0 = lds_addr(smem) + wid * 1024;  // (this wave's first piece)
  const Stager<DP> sk(a.k_row, a.dim, lane, wid), sv(a.v_row, a.dim, lane, wid);
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  if (kbeg < kend) {
    sk.all(kb_ + kbeg * a.k_row, lds0, word);
    sv.all(vb_ + kbeg * a.v_row, lds0 + TB, word);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
    const char* Kt = smem + buf * 2 * TB;
    const char* Vt = Kt + TB;
    dma_wait();
    __syncthreads();
    const uint64_t next = key_word(a.mask, loaded, n, k0 + BK);
    if (k0 + BK < kend) {
      const uint32_t to = lds0 + (buf ^ 1) * 2 * TB;
      sk.all(kb_ + (long long)(k0 + BK) * a.k_row, to, next);
      sv.all(vb_ + (long long)(k0 + BK) * a.v_row, to + TB, next);
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
    }
    const uint64_t now = word;
    word = next;
    if (q0 >= n || k0 > wlast + right || k0 + BK <= q0 - left || now == 0) continue;
    const bool edge = now != ~0ull || k0 < wlast - left || k0 + BK > q0 + right + 1;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = nd; }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows<DP>(Kt, kb * 32, c, lane), qf[c], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows<DP>(Vt, kb * 32, c, lane), df[c], dp, 0, 0, 0);
      }
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, nl)) * dp[r];
      if (edge) {
        const int base = k0 + kb * 32;
        const uint32_t see = (bits32(qi - left - base, qi + right + 1 - base) & (uint32_t)(now >> (kb * 32))) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = (see >> (8 * (r >> 2) + (r & 3))) & 1 ? ds[r] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x8 f = pack_acc(ds, j);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols<DP>(Kt, kb * 32 + j * 16, dt, lane), f, acc[dt], 0, 0, 0);
      }
    }
  }
  store_T<DP>(dq + (long long)(tile.row0 + qi) * a.dq_row + h * a.dq_head, acc, a.scale, a.dim, qi < n, half);
}

// dK, dV: 128 keys of one key head a workgroup, 32 a wave (lane = key), over the query heads of the group and tiles of 64 query rows
template <int DP>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void attn_gqa_dkv_kernel(const Args a, const uint16_t* __restrict__ dctx, const float* __restrict__ ndelta,
                                                              const float* __restrict__ nlse, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv,
                                                              int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) {
    const Gaps gap(a.seq_off, a.B, a.T);
    for (long long i = blockIdx.x; i < (long long)gap.count * a.kv_heads; i += gridDim.x)
      if (tid * 4 < a.dim) {
        const int row = gap.row((int)(i / a.kv_heads)), h = (int)(i % a.kv_heads);
        *reinterpret_cast<uint2*>(dk + row * a.dk_row + h * a.dk_head + tid * 4) = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(dv + row * a.dv_row + h * a.dv_head + tid * 4) = make_uint2(0u, 0u);
      }
  }
  const int G = a.heads / a.kv_heads, kvh = blockIdx.x % a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, blockIdx.x / a.kv_heads, lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int key0 = tile.first + wid * 32, kj = key0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(key0 + 31, n - 1);
  const int qbeg = max(tile.first - right, 0) & ~(BK - 1), qend = min(last + left + 1, n);
  const float sl2 = a.scale * kLog2e;
  const bool alive = kj < n && (!a.mask || a.mask[tile.row0 + kj] != 0);
  const bool all = __all(alive), none = !__any(alive);

  bf16x8 kf[DP / 16], vf[DP / 16];
  load_frags<DP>(kf, a.k + (long long)(tile.row0 + kj) * a.k_row + kvh * a.k_head, a.dim, alive, half);
  load_frags<DP>(vf, a.v + (long long)(tile.row0 + kj) * a.v_row + kvh * a.v_head, a.dim, alive, half);
  landed(kf);
  landed(vf);
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) { gk[dt][r] = 0.f; gv[dt][r] = 0.f; }

  constexpr int TB = BK * DP * 2, SB = 2 * TB + 2 * BK * 4;  // Q tile, dO tile, -lse and -delta of the rows
  const int tiles = qend > qbeg ? (qend - qbeg + BK - 1) / BK : 0, steps = tiles * G;
  const uint32_t lds0 = lds_addr(smem);
  const Stager<DP> sq(a.q_row, a.dim, lane, wid), sd(a.do_row, a.dim, lane, wid);
  auto fetch = [&](int i, uint32_t to) {
    const int h = kvh * G + i / tiles, q0 = qbeg + (i % tiles) * BK;
    const uint64_t rows = bits_below(n - q0);
    sq.all(a.q + (long long)(tile.row0 + q0) * a.q_row + h * a.q_head, to + wid * 1024, rows);
    sd.all(dctx + (long long)(tile.row0 + q0) * a.do_row + h * a.do_head, to + TB + wid * 1024, rows);
    if (wid < 2) {
      const rsrc_t rs = rsrc_of((wid == 0 ? nlse : ndelta) + (size_t)h * a.T + tile.row0 + q0, (uint32_t)min(n - q0, BK) * 4u);
      rsrc_settled(rs);
      dma4(rs, (uint32_t)lane * 4u, to + 2 * TB + wid * BK * 4);
    }
  };
  if (steps) fetch(0, lds0);
  for (int i = 0; i < steps; ++i) {
    const char* Qt = smem + (i & 1) * SB;
    const char* Dt = Qt + TB;
    const float* nl = reinterpret_cast<const float*>(Qt + 2 * TB);
    const float* nd = nl + BK;
    dma_wait();
    __syncthreads();
    if (i + 1 < steps) fetch(i + 1, lds0 + ((i + 1) & 1) * SB);
    const int q0 = qbeg + (i % tiles) * BK;
    if (none || q0 > wlast + left || q0 + BK <= key0 - right) continue;
    const bool edge = !all || q0 < wlast - right || q0 + BK > key0 + left + 1;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      f32x16 s, dp;
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const float4 d4 = *reinterpret_cast<const float4*>(nd + qb * 32 + 8 * rg + 4 * half);
        dp[rg * 4] = d4.x; dp[rg * 4 + 1] = d4.y; dp[rg * 4 + 2] = d4.z; dp[rg * 4 + 3] = d4.w;
        s[rg * 4] = s[rg * 4 + 1] = s[rg * 4 + 2] = s[rg * 4 + 3] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows<DP>(Qt, qb * 32, c, lane), kf[c], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows<DP>(Dt, qb * 32, c, lane), vf[c], dp, 0, 0, 0);
      }
      float p[16], ds[16];
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const float4 l4 = *reinterpret_cast<const float4*>(nl + qb * 32 + 8 * rg + 4 * half);
        const float ll[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) p[rg * 4 + e] = __builtin_amdgcn_exp2f(fmaf(s[rg * 4 + e], sl2, ll[e]));
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = p[r] * dp[r];
      if (edge) {
        const int base = q0 + qb * 32;
        const uint32_t see = alive ? bits32(kj - right - base, min(kj + left + 1, n) - base) >> (4 * half) : 0u;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool is = (see >> (8 * (r >> 2) + (r & 3))) & 1;
          p[r] = is ? p[r] : 0.f;
          ds[r] = is ? ds[r] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x8 pf = pack_acc(p, j), sf = pack_acc(ds, j);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          gv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols<DP>(Dt, qb * 32 + j * 16, dt, lane), pf, gv[dt], 0, 0, 0);
          gk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols<DP>(Qt, qb * 32 + j * 16, dt, lane), sf, gk[dt], 0, 0, 0);
        }
      }
    }
  }
  const long long row = tile.row0 + kj;
  store_T<DP>(dk + row * a.dk_row + kvh * a.dk_head, gk, a.scale, a.dim, kj < n, half);
  store_T<DP>(dv + row * a.dv_row + kvh * a.dv_head, gv, 1.0f, a.dim, kj < n, half);
}

// ------------------------------------------------------------------------------------------------ host
constexpr long long kMaxStride = 1ll << 23;  // elements: 64 rows of it stay inside a buffer descriptor's 31-bit offsets

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool stride_ok(long long row, long long head, int T, int heads) {  // (the stride of a single row or head is never used)
  return (T == 1 || (row >= 0 && row < kMaxStride && row % 8 == 0)) && (heads == 1 || (head >= 0 && head % 8 == 0));
}
// an output's rows must not overlap: heads inside a row's stride, or rows inside a head's
bool apart(long long row, long long head, int T, int heads, int D) {
  return (heads == 1 || head >= D) && (T == 1 || row >= D) && ((T == 1 || row >= (heads - 1) * head + D) || (heads == 1 || head >= (T - 1ll) * row + D));
}

int check(const Args* a, const char* what) {
  CK_ARG(a, "%s: null arguments", what);
  CK_ARG(a->q && a->k && a->v && a->seq_off, "%s: null pointer", what);
  CK_ARG(a->T > 0 && a->T < kFar && a->B > 0 && a->B < kFar, "%s: T=%d rows, B=%d sequences: 1 to 2^30 - 1 of each", what, a->T, a->B);
  CK_ARG(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0, "%s: heads=%d must be a multiple of kv_heads=%d", what, a->heads, a->kv_heads);
  CK_ARG(a->dim > 0 && a->dim <= 128 && a->dim % 8 == 0, "%s: head size %d must be a multiple of 8 up to 128", what, a->dim);
  CK_ARG(a->scale > 0.f && a->scale < INFINITY, "%s: scale must be positive and finite", what);
  CK_ARG(a->left >= -1 && a->right >= -1 && a->left < kFar && a->right < kFar, "%s: window (%d, %d): -1 (unlimited) or a number of rows", what, a->left, a->right);
  CK_ARG(aligned16(a->q) && aligned16(a->k) && aligned16(a->v), "%s: q, k, v must be 16-byte aligned", what);
  CK_ARG(stride_ok(a->q_row, a->q_head, a->T, a->heads) && stride_ok(a->k_row, a->k_head, a->T, a->kv_heads) && stride_ok(a->v_row, a->v_head, a->T, a->kv_heads), "%s: strides must be multiples of 8 elements, rows less than 2^23 apart", what);
  const long long units = ((long long)a->T / 128 + a->B) * a->heads;
  CK_ARG(units <= INT_MAX, "%s: too many rows and heads for one launch", what);
  return COCODR_OK;
}

bool long_rows(const Args* a) { return a->T / a->B >= 512; }
template <class K> void allow_lds(K kernel, int bytes) { (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); }
constexpr int kv_lds(int DP) { return 4 * BK * DP * 2; }
constexpr int kv3_lds(int DP) { return 6 * BK * DP * 2; }
constexpr int qd_lds(int DP) { return 2 * (2 * BK * DP * 2 + 2 * BK * 4); }
void lds_limits() {
  static cocodr_lds_once once;
  if (!once.pending()) return;
  allow_lds(attn_gqa_fwd2_kernel<64>, kv3_lds(64)); allow_lds(attn_gqa_fwd2_kernel<128>, kv3_lds(128));
  allow_lds(attn_gqa_fwd_kernel<64>, kv_lds(64)); allow_lds(attn_gqa_fwd_kernel<128>, kv_lds(128));
  allow_lds(attn_gqa_dq_kernel<64>, kv_lds(64)); allow_lds(attn_gqa_dq_kernel<128>, kv_lds(128));
  allow_lds(attn_gqa_dkv_kernel<64>, qd_lds(64)); allow_lds(attn_gqa_dkv_kernel<128>, qd_lds(128));
  once.done();
}

}  // namespace

extern "C" int cocodr_attn_gqa_fwd(const cocodr_attn_gqa_args* a, uint16_t* ctx, float* lse, int fill, cocodr_stream_t stream) {
  if (int rc = check(a, "attn_gqa_fwd")) return rc;
  CK_ARG(ctx && lse && aligned16(ctx), "attn_gqa_fwd: ctx and lse must be given, ctx 16-byte aligned");
  CK_ARG(stride_ok(a->o_row, a->o_head, a->T, a->heads) && apart(a->o_row, a->o_head, a->T, a->heads, a->dim), "attn_gqa_fwd: ctx strides must be multiples of 8 and keep its rows apart");
  lds_limits();
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((a->T / 128 + a->B) * a->heads));
  if (long_rows(a)) {
    const dim3 grid2((unsigned)((a->T / 256 + a->B) * a->heads));
    if (a->dim <= 64) hipLaunchKernelGGL(attn_gqa_fwd2_kernel<64>, grid2, dim3(256), kv3_lds(64), st, *a, ctx, lse, fill);
    else hipLaunchKernelGGL(attn_gqa_fwd2_kernel<128>, grid2, dim3(256), kv3_lds(128), st, *a, ctx, lse, fill);
  } else if (a->dim <= 64) hipLaunchKernelGGL(attn_gqa_fwd_kernel<64>, grid, dim3(256), kv_lds(64), st, *a, ctx, lse, fill);
  else hipLaunchKernelGGL(attn_gqa_fwd_kernel<128>, grid, dim3(256), kv_lds(128), st, *a, ctx, lse, fill);
  CK_LAUNCH("attn_gqa_fwd");
  return COCODR_OK;
}

extern "C" size_t cocodr_attn_gqa_bwd_workspace_floats(const cocodr_attn_gqa_args* a) { return a && a->T > 0 && a->heads > 0 ? (size_t)2 * a->T * a->heads : 0; }

extern "C" int cocodr_attn_gqa_bwd(const cocodr_attn_gqa_args* a, const uint16_t* ctx, const uint16_t* dctx, const float* lse, uint16_t* dq,
                                   uint16_t* dk, uint16_t* dv, int fill, float* workspace, size_t workspace_floats, cocodr_stream_t stream) {
  if (int rc = check(a, "attn_gqa_bwd")) return rc;
  CK_ARG(ctx && dctx && lse && dq && dk && dv, "attn_gqa_bwd: null pointer");
  CK_ARG(aligned16(ctx) && aligned16(dctx) && aligned16(dq) && aligned16(dk) && aligned16(dv), "attn_gqa_bwd: tensors must be 16-byte aligned");
  CK_ARG(stride_ok(a->o_row, a->o_head, a->T, a->heads) && stride_ok(a->do_row, a->do_head, a->T, a->heads), "attn_gqa_bwd: strides must be multiples of 8 elements, rows less than 2^23 apart");
  CK_ARG(stride_ok(a->dq_row, a->dq_head, a->T, a->heads) && apart(a->dq_row, a->dq_head, a->T, a->heads, a->dim) && stride_ok(a->dk_row, a->dk_head, a->T, a->kv_heads) &&
             apart(a->dk_row, a->dk_head, a->T, a->kv_heads, a->dim) && stride_ok(a->dv_row, a->dv_head, a->T, a->kv_heads) && apart(a->dv_row, a->dv_head, a->T, a->kv_heads, a->dim),
         "attn_gqa_bwd: gradient strides must be multiples of 8 and keep the rows apart");
  if (!workspace || workspace_floats < cocodr_attn_gqa_bwd_workspace_floats(a)) {
    cocodr_set_error("attn_gqa_bwd: workspace of %zu floats is too small", workspace_floats);
    return COCODR_ERR_WORKSPACE;
  }
  lds_limits();
  hipStream_t st = (hipStream_t)stream;
  float *ndelta = workspace, *nlse = workspace + (size_t)a->T * a->heads;
  const dim3 gq((unsigned)((a->T / 128 + a->B) * a->heads)), gk((unsigned)((a->T / 128 + a->B) * a->kv_heads));
  if (a->dim <= 64) {
    hipLaunchKernelGGL(attn_gqa_dq_kernel<64>, gq, dim3(256), kv_lds(64), st, *a, ctx, dctx, lse, ndelta, nlse, dq, fill);
    hipLaunchKernelGGL(attn_gqa_dkv_kernel<64>, gk, dim3(256), qd_lds(64), st, *a, dctx, ndelta, nlse, dk, dv, fill);
  } else {
    hipLaunchKernelGGL(attn_gqa_dq_kernel<128>, gq, dim3(256), kv_lds(128), st, *a, ctx, dctx, lse, ndelta, nlse, dq, fill);
    hipLaunchKernelGGL(attn_gqa_dkv_kernel<128>, gk, dim3(256), qd_lds(128), st, *a, dctx, ndelta, nlse, dk, dv, fill);
  }
  CK_LAUNCH("attn_gqa_bwd");
  return COCODR_OK;
}
