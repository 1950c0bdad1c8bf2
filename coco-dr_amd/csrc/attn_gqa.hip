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
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "common.h"
#include "prof.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Where a running maximum starts: finite, so that a row without any key gives exp2(-inf - kLow) = 0 and no NaN, and far below every score that fp32
// can subtract from another (up to 2^24 or so; a row of scores below kLow would pass for one without keys).
constexpr float kLow = -1e30f;
// A running maximum that is outgrown by less than 2^kGrow is left as it is: terms of up to 2^kGrow are as exact in fp32 and bf16 as those below 1, and
// the accumulators are at most 2^kGrow times a sum of |v|: finite below 2^108.
constexpr float kGrow = 20.0f;
constexpr int kFar = 1 << 30;   // an unlimited window; i + kFar stays inside an int for every row index < 2^30
constexpr int BK = 64;          // rows of a staged tile

typedef cocodr_attn_gqa_args Args;

// f(0), f(1), .. f(N - 1) with the index as a constant
template <int N, class F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}
#define SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)

// ------------------------------------------------------------------------------------------------ tiles in LDS
// [rows][DP] bf16, DP = 64 or 128 (the head size rounded up; columns behind it are zeros).  The 16-byte chunks of a row are permuted
// so that both reads are free of bank conflicts: ds_read_b128 of 16 consecutive rows at one chunk, and the transposing read of 4
// consecutive rows x 4 chunks.
template <int DP> __device__ __forceinline__ int swz(int row) {
  if constexpr (DP == 64) return swz64(row);
  else return ((row & 3) << 2) | ((row >> 2) & 3);
}
template <int DP> __device__ __forceinline__ int tile_off(int row, int ch) { return row * (DP * 2) + ((ch ^ swz<DP>(row)) << 4); }

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
template <class V> __device__ __forceinline__ LDS_PTR(V) lds_at(uint32_t addr) { return (LDS_PTR(V))(uintptr_t)addr; }
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(LDS_PTR(const void))p; }
__device__ __forceinline__ void dma16(rsrc_t rs, uint32_t off, uint32_t more, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(rs), "s"(more), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void dma4(rsrc_t rs, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(rs), "s"(dst) : "memory", "m0");
}
// this wave's transfers are in LDS; with the barrier behind it, every wave's
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// the lane's number, made where it is used: kept in a register, or what is derived from it, it is one too many in the kernels that use them all
__device__ __forceinline__ int fresh_lane() {
  int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(l));
  return l;
}

// BK rows of one head into a tile by LDS DMA: a wave's instruction (a piece) writes 1 KiB lane-linear, so the permutation goes into the source
// addresses.  Rows whose bit of `rows` is 0 (behind the sequence, masked out) and columns >= D are addressed behind the descriptor's
// end and arrive as zeros: whatever stands there in memory, NaN too, is not read.  The descriptor reaches over one tile only, so its
// 32-bit offsets do for any buffer.  Wave w of 4 has the pieces w, w + 4, ..: the permutation of its rows is the same in each, and a piece's
// offset differs from the first's by a scalar.
template <int DP> struct Stager {
  static constexpr int CH = DP / 8, RP = 64 / CH, PIECES = BK / RP / 4;  // chunks of a row, rows of a piece, pieces of a wave
  uint32_t ldb, span, first;  // bytes of a row, of a tile; this lane's offset in its wave's first piece
  int wid, D;
  __device__ __forceinline__ Stager(long long ld, int D_, int lane, int wid_) : wid(wid_), D(D_) {
    ldb = (uint32_t)ld * 2u;
    span = (uint32_t)(BK - 1) * ldb + (uint32_t)D * 2u;
    first = first_of(lane);
  }
  __device__ __forceinline__ uint32_t first_of(int lane) const {
    const int row = wid * RP + lane / CH, ch = (lane & (CH - 1)) ^ swz<DP>(row);
    return ch * 8 < D ? (uint32_t)row * ldb + (uint32_t)ch * 16u : 0x80000000u;
  }
  __device__ __forceinline__ rsrc_t tile(const uint16_t* src) const { return rsrc_of(src, span); }
  __device__ __forceinline__ uint32_t more(int i) const { return (uint32_t)(i * 4 * RP) * ldb; }  // piece i's offset behind the first's
  // all pieces; dst: the wave's first piece of the tile in LDS
  __device__ __forceinline__ void all(const uint16_t* src, uint32_t dst, uint64_t rows) const {
    const rsrc_t rs = tile(src);
    rsrc_settled(rs);
    if (rows == ~0ull) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) dma16(rs, first, more(i), dst + i * 4096);
    } else {
      const int row = wid * RP + fresh_lane() / CH;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) dma16(rs, (rows >> (row + i * 4 * RP)) & 1 ? first : 0x80000000u, more(i), dst + i * 4096);
    }
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
// The tiles of TILE rows are numbered without a table, and a launch has T / TILE + B workgroups, at least as many as there are tiles.
//   up to 256 sequences: consecutive numbers in the order of the rows, from a sum over the sequences that every wave makes, four a lane; the numbers
//     that no tile has come last, where they hold nobody up (64 x 128 rows, 12 heads, forward and backward: 58 us; 75 with the numbers below, every
//     second of which is empty there; forward of 256 sequences of 20 to 256, 16 heads, 70 us, of 257 with the numbers below 75, of 512 145)
//   more: tile t of sequence b has the number off[b] / TILE + b + t - rounding down and the + b leave a sequence at least as many numbers as it has
//     tiles -, and number -> sequence is the last b with off[b] / TILE + b <= number: a search 64 wide
// When sequences are long and few, the numbers go by the work of a tile instead, the most first: a workgroup with much to do that starts
// among the last is waited for by an empty chip.  A lane then has a sequence of c tiles.
//   kUp, kDown: the work grows (falls) along a sequence, so tile x (tile c - 1 - x) of every sequence that has it comes before tile x - 1:
//     x is the largest with S(x) = sum max(c - x, 0) > number, found 64 candidates at a time
//   kLevel: it is the same along a sequence: all tiles of the longest sequence, then of the next
struct Tile {
  int n, first, row0;  // the sequence's rows (0: nothing to do), this tile's first row in it, the sequence's first row in the buffer
};
enum Order { kPlain, kUp, kDown, kLevel };
__device__ __forceinline__ int tiles_from(int c, int B, int x) {  // S(x); x may differ from lane to lane
  int sum = 0;
  for (int b = 0; b < B; ++b) sum += max(__builtin_amdgcn_readlane(c, b) - x, 0);
  return sum;
}
template <int TILE> __device__ __forceinline__ Tile find_tile(const int32_t* off, int B, int T, int num, int order, int lane) {
  int lo = 0, n = B, t = -1;
  if (order == kPlain && B <= 256) {
    const int per = (B + 63) >> 6;
    int at[5], c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i) at[i] = off[min(lane * per + i, B)];  // (all five always: a condition would have them wait for one another)
#pragma unroll
    for (int i = 0; i < 5; ++i) at[i] = min(max(at[i], 0), T);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = i < per ? (max(at[i + 1] - at[i], 0) + TILE - 1) / TILE : 0;
      sum += c[i];
    }
    int upto = sum;  // the tiles of this lane's sequences and of those before
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x142, 0xa, 0xf, false);  // the last lane of each row of 16 to the next row
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
    const uint64_t found = __ballot(num < upto && num >= upto - sum);
    if (found == 0) return Tile{0, 0, 0};
    int t = num - (upto - sum), a = at[0], e = at[1];
    bool there = t < c[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      t -= there ? 0 : c[i - 1];
      a = there ? a : at[i];
      e = there ? e : at[i + 1];
      there = there || t < c[i];
    }
    const int from = __builtin_amdgcn_readfirstlane(__ffsll((long long)found) - 1);
    a = __builtin_amdgcn_readlane(a, from);
    return Tile{__builtin_amdgcn_readlane(e, from) - a, __builtin_amdgcn_readlane(t, from) * TILE, a};
  }
  if (order == kPlain) {
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
  } else {
    int c = 0;
    if (lane < B) {
      const int a = min(max(off[lane], 0), T);
      c = (min(max(off[lane + 1], a), T) - a + TILE - 1) / TILE;
    }
    bool here;
    if (order == kLevel) {
      int start = 0;
      for (int b = 0; b < B; ++b) {
        const int other = __builtin_amdgcn_readlane(c, b);
        start += other > c || (other == c && b < lane) ? other : 0;
      }
      t = num - start;
      here = t >= 0 && t < c;
    } else {
      int x = 0, span = T / TILE + 1;
      while (span > 1) {
        const int step = (span + 63) >> 6;
        const bool more = lane * step < span && tiles_from(c, B, x + lane * step) > num;
        const int cut = max(__builtin_amdgcn_readfirstlane((int)__popcll(__ballot(more))) - 1, 0) * step;
        span = min(step, span - cut);
        x += cut;
      }
      const uint64_t have = __ballot(c > x);
      here = c > x && (int)__popcll(have & ((1ull << lane) - 1)) == num - tiles_from(c, B, x + 1);
      t = order == kUp ? x : c - 1 - x;
    }
    const uint64_t found = __ballot(here);
    if (found == 0) return Tile{0, 0, 0};
    lo = __ffsll((long long)found) - 1;
    t = __builtin_amdgcn_readlane(t, __builtin_amdgcn_readfirstlane(lo));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int a = min(max(off[lo], 0), T), e = min(max(off[lo + 1], a), T);
  if (order == kPlain) t = num - (a / TILE + lo);
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

// v where bit AT of `see` is set, -inf where it is not: two instructions (hipcc's own choice is a test, a wait state and a selection, 40 % of a
// masked tile's instructions)
template <int AT> __device__ __forceinline__ float seen(uint32_t see, float v) {
  uint32_t all;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(all) : "v"(see), "n"(AT));
  return __uint_as_float((__float_as_uint(v) & all) | (__float_as_uint(-INFINITY) & ~all));
}

// which of the BK keys from k0 on exist and are not masked out.  The load is started (key_word_load) one tile before its ballot is taken.
__device__ __forceinline__ int key_word_load(const int32_t* mask, int row0, int n, int k0, int lane) {
  return mask && k0 + lane < n ? mask[row0 + k0 + lane] : 1;
}
__device__ __forceinline__ uint64_t key_word(const int32_t* mask, int loaded, int n, int k0) {
  const uint64_t w = bits_below(n - k0);
  return mask ? w & __ballot(loaded != 0) : w;
}

// LDS addresses of the operand fragments of tiles: row(c) has rows lane & 31 of the 32 at AT, contraction columns 16 c + 8 (lane >> 5) .. + 7;
// col(dt) is of the transposed tile: output row = column 32 dt + (lane & 31), contraction = tile rows 4 (lane >> 5) + {0..3} and + 8 behind AT, the rows
// that accumulator registers 8 j .. 8 j + 7 of a 32 x 32 product hold (AT = row 16 j).  Here all of them in registers for the whole loop: what
// differs from use to use is an offset in the instruction.
template <int DP> struct Frags {
  uint32_t rows[DP / 16], cols[DP / 16];  // of row fragments 0, 1, .. and of column fragments (dt, rows 0 / 8) of a tile
  __device__ __forceinline__ Frags(uint32_t at, int lane) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      rows[i] = at + tile_off<DP>(lane & 31, 2 * i + (lane >> 5));
      const int col = (i >> 1) * 32 + ((g & 1) << 4) + ((c & 3) << 2), row = ((g >> 1) << 2) + (c >> 2) + (i & 1) * 8;
      cols[i] = at + tile_off<DP>(row, col >> 3) + ((col & 7) << 1);
    }
  }
  __device__ __forceinline__ void forget() {}
  template <int AT> __device__ __forceinline__ bf16x8 row(int c) const { return *lds_at<const bf16x8>(rows[c] + AT); }
  template <int AT> __device__ __forceinline__ bf16x8 col(int dt) const {
    return join_tr(__builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(cols[2 * dt] + AT)),
                   __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(cols[2 * dt + 1] + AT)));
  }
};

// The same addresses as that of fragment 0 with a few bits flipped: a tile's rows start at multiples of DP * 2 bytes, so the chunk
// number and its permutation are address bits of their own, and one register and an exclusive or do for eight.
template <int DP> struct Bits {
  uint32_t rows, cols;
  __device__ __forceinline__ Bits(uint32_t at, int lane) {
    const int g = lane >> 4, c = lane & 15, col = ((g & 1) << 4) + ((c & 3) << 2), row = ((g >> 1) << 2) + (c >> 2);
    rows = at + tile_off<DP>(lane & 31, lane >> 5);
    cols = at + tile_off<DP>(row, col >> 3) + ((col & 7) << 1);
  }
  // what they are is forgotten: or hipcc makes the flipped addresses once, in front of the loop, and keeps each in a register of its own
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(rows), "+v"(cols)); }
  template <int AT> __device__ __forceinline__ bf16x8 row(int c) const { return *lds_at<const bf16x8>((rows ^ (c << 5)) + AT); }
  // rows + 8 flip bit 1 of the permutation (DP = 128: row bit 3 is its bit 1; DP = 64: row bit 3 its bit 1, too)
  template <int AT> __device__ __forceinline__ bf16x8 col(int dt) const {
    return join_tr(__builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>((cols ^ (dt << 6)) + AT)),
                   __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>((cols ^ ((dt << 6) | 32)) + AT + 8 * DP * 2)));
  }
};

// ------------------------------------------------------------------------------------------------ forward
__device__ __forceinline__ void fill_gaps(const Args& a, uint16_t* ctx, float* lse, int tid) {
  const Gaps gap(a.seq_off, a.B, a.T);
  for (long long i = blockIdx.x; i < (long long)gap.count * a.heads; i += gridDim.x) {
    const int row = gap.row((int)(i / a.heads)), h = (int)(i % a.heads);
    if (tid * 4 < a.dim) *reinterpret_cast<uint2*>(ctx + row * a.o_row + h * a.o_head + tid * 4) = make_uint2(0u, 0u);
    if (tid == 0) lse[(size_t)h * a.T + row] = -INFINITY;
  }
}

// A workgroup has 128 query rows of one head, each of its four waves 32 of them; K and V pass through LDS in tiles of 64 keys, two tiles each, so that
// a tile is on its way while the one before is worked on.  Scores, statistics and the output never leave the registers: one pass over the keys.
// Heads of 128, long sequences: bound by the matrix pipe, and that by power: 8192 causal, 32 / 8 heads, 566 us = 971 TFLOP/s, where the pipe is 48 % busy
// at 1.9 GHz; 64 rows a wave (one wave a SIMD, half the LDS traffic) took 580 us at 2.4 GHz, eight waves sharing a tile 571.  So 32 rows and two
// workgroups a CU, which short sequences want too (129 against 84 us with eight waves, 256 sequences of 20 to 256).
// Heads of 64, short sequences: bound by what stands before the first product - offsets, mask, first tile, each waiting for the one before, 5 of a
// workgroup's 10 us - so as many workgroups at once as registers allow (122: four a CU; addresses by flipped bits instead of a register each): 256
// sequences of 20 to 256, 16 heads, masked: 70 us, 2.8 TB/s.  Two heads after one another in a workgroup saved nothing (71 - 75 us).
template <int DP>
__global__ __launch_bounds__(256, DP == 64 ? 4 : 2) void attn_gqa_fwd_kernel(const Args a, uint16_t* __restrict__ ctx, float* __restrict__ lse, int order, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) fill_gaps(a, ctx, lse, tid);
  const int G = a.heads / a.kv_heads;
  const int unit = blockIdx.x % a.heads, kvh = unit % a.kv_heads, h = kvh * G + unit / a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, blockIdx.x / a.heads, order, lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int q0 = tile.first + wid * 32, qi = q0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(q0 + 31, n - 1);
  const int kbeg = max(tile.first - left, 0) & ~(BK - 1), kend = min(last + right + 1, n);
  const int wbeg = max(q0 - left, 0), wend = q0 < n ? min(wlast + right + 1, n) : 0;  // the keys that this wave's rows see
  const int allbeg = wlast - left, allend = q0 + right + 1;                           // ... that all of them see
  const uint16_t* ks = a.k + (long long)(tile.row0 + kbeg) * a.k_row + kvh * a.k_head;  // the tile that is sent for next
  const uint16_t* vs = a.v + (long long)(tile.row0 + kbeg) * a.v_row + kvh * a.v_head;
  const float sl2 = a.scale * kLog2e;

  constexpr int TB = BK * DP * 2, NC = DP / 16, ND = DP / 32;
  const uint32_t mine = lds_addr(smem) + wid * 1024;  // (this wave's first piece)
  const Stager<DP> sk(a.k_row, a.dim, lane, wid), sv(a.v_row, a.dim, lane, wid);
  bf16x8 qf[NC];
  load_frags<DP>(qf, a.q + (long long)(tile.row0 + qi) * a.q_row + h * a.q_head, a.dim, qi < n, half);
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  sk.all(ks, mine, word);
  sv.all(vs, mine + TB, word);

  f32x16 o[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = kLow, l = 0.f;
  std::conditional_t<DP == 64, Bits<DP>, Frags<DP>> f(lds_addr(smem), lane);
  landed(qf);

  // one tile of keys from k0, in buffer BUF
  auto work = [&](auto buf_, int k0) {
    constexpr int BUF = decltype(buf_)::value, KA = BUF * 2 * TB, VA = KA + TB;
    dma_wait();
    __syncthreads();
    const uint64_t now = word;
    if (k0 + BK < kend) {
      word = key_word(a.mask, loaded, n, k0 + BK);
      const uint32_t to = mine + (BUF ^ 1) * 2 * TB;
      ks += BK * a.k_row;
      vs += BK * a.v_row;
      sk.all(ks, to, word);
      sv.all(vs, to + TB, word);
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
    }
    if (k0 >= wend || k0 + BK <= wbeg) return;
    f.forget();
    f32x16 s[2];
    bf16x8 f0[NC], f1[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) f0[c] = f.template row<KA>(c);
    SCHED_FENCE();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f1[c] = f.template row<KA + TB / 2>(c);
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f0[c], qf[c], s[0], 0, 0, 0);
      SCHED_FENCE();
    }
    bf16x8 vf[ND];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c % 2 == 0) vf[c / 2] = f.template col<VA>(c / 2);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f1[c], qf[c], s[1], 0, 0, 0);
      SCHED_FENCE();
    }
    if (now != ~0ull || k0 < allbeg || k0 + BK > allend) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int base = k0 + kb * 32;
        const uint32_t see = (bits32(qi - left - base, qi + right + 1 - base) & (uint32_t)(now >> (kb * 32))) >> (4 * half);
        each<16>([&](auto r_) {
          constexpr int r = decltype(r_)::value;
          s[kb][r] = seen<8 * (r >> 2) + (r & 3)>(see, s[kb][r]);
        });
      }
    }
    const float top = max_halves(max32(s)) * sl2;
    if (__any(top > m + kGrow)) {
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      if (__any(l != 0.f)) {  // (or the sums are zeros: nothing to scale)
        l *= f;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= f;
      }
    }
    // P of a 16-key step is made while the products of the step before run; the step's rows of V are fetched one step ahead
    each<4>([&](auto t_) {
      constexpr int t = decltype(t_)::value;
      float p[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[t >> 1][(t & 1) * 8 + r], sl2, -m));
        l += p[r];
      }
      const bf16x8 pf = as_bf16x8(pack8(p));
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[dt], pf, o[dt], 0, 0, 0);
        if constexpr (t < 3) vf[dt] = f.template col<VA + (t + 1) * 16 * DP * 2>(dt);
      }
    });
  };
  for (int k0 = kbeg; k0 < kend; k0 += 2 * BK) {
    work(std::integral_constant<int, 0>{}, k0);
    if (k0 + BK < kend) work(std::integral_constant<int, 1>{}, k0 + BK);
  }
  l = sum_halves(l);
  if (qi < n && lane < 32) lse[(size_t)h * a.T + tile.row0 + qi] = l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
  store_T<DP>(ctx + (long long)(tile.row0 + qi) * a.o_row + h * a.o_head, o, l > 0.f || l != l ? 1.0f / l : 0.f, a.dim, qi < n, half);
}

// ------------------------------------------------------------------------------------------------ backward
// how many keys row i of a sequence sees, masked ones among them
__device__ __forceinline__ int keys_of(int i, int n, int left, int right) { return min(i + right, n - 1) - max(i - left, 0) + 1; }

// dQ: 128 query rows of one head a workgroup, 32 a wave (lane = query), over tiles of 64 keys as in the forward.  A wave has its rows of dO in
// registers: with ctx beside them it also makes -delta and -lse (in log2 units) of its rows and leaves them, [heads][T] each, for the dK / dV kernel.
// ctx is rounded to bf16, and so is off by 2^-9 of itself, rms, against dP of which it is the mean: nothing beside the rounding of dS where a row sees
// many keys, but up to twice its effect where it sees a few.  Workgroups with a row that reaches up to 64 keys (masked ones counted) take delta = sum p dp
// from a pass of their own over their few tiles instead of from ctx (16 sequences of 1 to 2048: dq off by 2.4e-3 in norm, 2.6e-3 with ctx; short ones
// alone 2.3e-3 and 4e-3).  What the pass costs, forward and backward, 12 heads of 64: 3 sequences of 2047 to 4099 with windows of 16 + 16 82 us against
// 74, 32 + 32 77 against 74; 256 causal sequences of 1 to 64 69 against 65; the 16 of 1 to 2048 and whole long ones nothing.
// 4 x 4096 causal, 32 / 8 heads of 128: 765 - 830 us, 3 products of 275 GFLOP, 1.0 PFLOP/s: power again.  64 x 128, 12 heads of 64: 20 us, 76 MB at 3.8 TB/s.
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_gqa_dq_kernel(const Args a, const uint16_t* __restrict__ ctx, const uint16_t* __restrict__ dctx,
                                                             const float* __restrict__ lse, float* __restrict__ ndelta, float* __restrict__ nlse,
                                                             uint16_t* __restrict__ dq, int order, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) {
    const Gaps gap(a.seq_off, a.B, a.T);
    for (long long i = blockIdx.x; i < (long long)gap.count * a.heads; i += gridDim.x)
      if (tid * 4 < a.dim) *reinterpret_cast<uint2*>(dq + gap.row((int)(i / a.heads)) * a.dq_row + (int)(i % a.heads) * a.dq_head + tid * 4) = make_uint2(0u, 0u);
  }
  const int G = a.heads / a.kv_heads;
  const int unit = blockIdx.x % a.heads, kvh = unit % a.kv_heads, h = kvh * G + unit / a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, blockIdx.x / a.heads, order, lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int q0 = tile.first + wid * 32, qi = q0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(q0 + 31, n - 1);
  const int kbeg = max(tile.first - left, 0) & ~(BK - 1), kend = min(last + right + 1, n);
  const int wbeg = max(q0 - left, 0), wend = q0 < n ? min(wlast + right + 1, n) : 0;  // (as in the forward)
  const int allbeg = wlast - left, allend = q0 + right + 1;
  const uint16_t *ks, *vs;
  const float sl2 = a.scale * kLog2e;
  constexpr int TB = BK * DP * 2, NC = DP / 16, ND = DP / 32;

  bf16x8 qf[DP / 16], df[DP / 16];
  load_frags<DP>(qf, a.q + (long long)(tile.row0 + qi) * a.q_row + h * a.q_head, a.dim, qi < n, half);
  load_frags<DP>(df, dctx + (long long)(tile.row0 + qi) * a.do_row + h * a.do_head, a.dim, qi < n, half);
  const size_t at = (size_t)h * a.T + tile.row0 + qi;
  // (an empty row's lse is -inf: its probabilities are exp2(s - inf) = 0, whatever s is)
  float nl = qi < n ? (lse[at] == -INFINITY ? -INFINITY : -lse[at] * kLog2e) : 0.f;
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(nl));
  float nd = 0.f;
  const int few = min(keys_of(tile.first, n, left, right), keys_of(last, n, left, right));
  if (few > 64) {
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
  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

  const uint32_t lds0 = lds_addr(smem) + wid * 1024;  // (this wave's first piece)
  const Stager<DP> sk(a.k_row, a.dim, lane, wid), sv(a.v_row, a.dim, lane, wid);
  int loaded;
  uint64_t word;
  auto first_tile = [&]() {
    loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
    word = key_word(a.mask, loaded, n, kbeg);
    loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
    ks = a.k + (long long)(tile.row0 + kbeg) * a.k_row + kvh * a.k_head;
    vs = a.v + (long long)(tile.row0 + kbeg) * a.v_row + kvh * a.v_head;
    sk.all(ks, lds0, word);
    sv.all(vs, lds0 + TB, word);
  };
  first_tile();
  float sum = 0.f;
  Bits<DP> f(lds_addr(smem), lane);
  // one tile of keys from k0, in buffer BUF; DELTA: only its share of delta
  auto work = [&](auto buf_, auto delta_, int k0) {
    constexpr int BUF = decltype(buf_)::value;
    constexpr bool DELTA = decltype(delta_)::value;
    dma_wait();
    __syncthreads();
    const uint64_t now = word;
    if (k0 + BK < kend) {
      word = key_word(a.mask, loaded, n, k0 + BK);
      const uint32_t to = lds0 + (BUF ^ 1) * 2 * TB;
      ks += BK * a.k_row;
      vs += BK * a.v_row;
      sk.all(ks, to, word);
      sv.all(vs, to + TB, word);
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
    }
    if (k0 >= wend || k0 + BK <= wbeg) return;
    const bool edge = now != ~0ull || k0 < allbeg || k0 + BK > allend;
    each<2>([&](auto kb_) {
      // (fragments are read DEEP - 1 ahead of their products)
      constexpr int kb = decltype(kb_)::value, K = BUF * 2 * TB + kb * TB / 2, V = K + TB, DEEP = 3;
      // (none of these 32 is seen: 1 % of 4 x 4096 causal with heads of 128.  With heads of 64 the branch costs 64 x 128 rows as much as it saves a window.)
      if (DP == 128 && (k0 + kb * 32 >= wend || k0 + kb * 32 + 32 <= wbeg)) return;
      f.forget();
      f32x16 s, dp;
      bf16x8 x[DEEP], z[DEEP];
      SCHED_FENCE();
#pragma unroll
      for (int c = 0; c < DEEP - 1; ++c) x[c] = f.template row<K>(c);
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = DELTA ? 0.f : nd; }  // dP starts at -delta
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        SCHED_FENCE();
        const int u = c + DEEP - 1;
        x[u % DEEP] = u < NC ? f.template row<K>(u) : f.template row<V>(u - NC);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[c % DEEP], qf[c], s, 0, 0, 0);
      }
      SCHED_FENCE();
      if (edge) {
        const int base = k0 + kb * 32;
        const uint32_t see = (bits32(qi - left - base, qi + right + 1 - base) & (uint32_t)(now >> (kb * 32))) >> (4 * half);
        each<16>([&](auto r_) {
          constexpr int r = decltype(r_)::value;
          s[r] = seen<8 * (r >> 2) + (r & 3)>(see, s[r]);
        });
      }
      // beside the products of dP: the probabilities
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        SCHED_FENCE();
        const int u = c + DEEP - 1;
        if (u < NC) x[(NC + u) % DEEP] = f.template row<V>(u);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[(NC + c) % DEEP], df[c], dp, 0, 0, 0);
#pragma unroll
        for (int e = c * 16 / NC; e < (c + 1) * 16 / NC; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], sl2, nl));
      }
      SCHED_FENCE();
      if constexpr (DELTA) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sum = fmaf(s[e], dp[e], sum);
        return;
      }
      each<DEEP - 1>([&](auto k) { z[decltype(k)::value] = f.template col<K + decltype(k)::value / ND * 16 * DP * 2>(decltype(k)::value % ND); });
      bf16x8 pf[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = s[j * 8 + e] * dp[j * 8 + e];
        pf[j] = as_bf16x8(pack8(d));
      }
      each<2 * ND>([&](auto k_) {
        constexpr int k = decltype(k_)::value, u = k + DEEP - 1;
        SCHED_FENCE();
        if constexpr (u < 2 * ND) z[u % DEEP] = f.template col<K + u / ND * 16 * DP * 2>(u % ND);
        acc[k % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z[k % DEEP], pf[k / ND], acc[k % ND], 0, 0, 0);
      });
      SCHED_FENCE();
    });
  };
  auto pass = [&](auto delta) {
    for (int k0 = kbeg; k0 < kend; k0 += 2 * BK) {
      work(std::integral_constant<int, 0>{}, delta, k0);
      if (k0 + BK < kend) work(std::integral_constant<int, 1>{}, delta, k0 + BK);
    }
  };
  if (few <= 64) {
    pass(std::true_type{});
    nd = -sum_halves(sum);
    __syncthreads();
    first_tile();
  }
  if (qi < n && lane < 32) {
    ndelta[at] = nd;
    nlse[at] = nl;
  }
  pass(std::false_type{});
  store_T<DP>(dq + (long long)(tile.row0 + qi) * a.dq_row + h * a.dq_head, acc, a.scale, a.dim, qi < n, half);
}

// the tiles of queries that see a tile of 128 keys, and in how many parts a group's heads are summed for it
__device__ __forceinline__ int query_tiles(const Args& a, const Tile& t) {
  const int beg = max(t.first - (a.right < 0 ? kFar : a.right), 0) & ~(BK - 1);
  const int end = min(min(t.first + 127, t.n - 1) + (a.left < 0 ? kFar : a.left) + 1, t.n);
  return end > beg ? (end - beg + BK - 1) / BK : 0;
}
// In how many parts a tile's steps (tiles of 64 queries, of every head of the group) are summed: `split` is the most, a power of two, `part` the steps that
// a part has to have more than.
struct Split { int split, part; };
__device__ __forceinline__ int parts_of(int steps, Split s) {
  int n = s.split;
  while (n > 1 && steps <= s.part * n) n >>= 1;
  return n;
}

// dK, dV: 128 keys of one key head a workgroup, 32 a wave (lane = key), over the query heads of the group and tiles of 64 query rows.  The wave's
// K and V fragments and its 128 accumulators stay in registers: 256 of them are just enough, and leave room for a second wave on the SIMD.  The second
// wave is what it takes: alone on its SIMD a wave issues an instruction every 4.8 clocks and waits 8 for a result, and the kernel took 1561 us for
// 4 x 4096 causal, 32 / 8 heads of 128; with two it takes 1010 - 1094, 4 products of 275 GFLOP, 1.05 PFLOP/s.  What it costs: addresses made by flipping
// bits, fragments fetched two products ahead and not more, three of K's in LDS, the probabilities two registers at a time beside dP's products.
// 64 x 128, 12 heads of 64: 21 us, 76 MB at 3.6 TB/s.  (One kernel for dQ, dK and dV of such short sequences, dS through LDS: 31 us + 4 for the
// other's empty launch, against 20 + 21; with registers for it, windows over long sequences lost as much as it won.)
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_gqa_dkv_kernel(const Args a, const uint16_t* __restrict__ dctx, const float* __restrict__ ndelta,
                                                              const float* __restrict__ nlse, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv,
                                                              f32x4* __restrict__ part, Split split, int order, int fill) {
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
  const int kvh = blockIdx.x % a.kv_heads, sub = blockIdx.x / a.kv_heads % split.split, num = blockIdx.x / (a.kv_heads * split.split);
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, num, order, lane);
  if (tile.n == 0) return;
  const int n = tile.n, left = a.left < 0 ? kFar : a.left, right = a.right < 0 ? kFar : a.right;
  const int key0 = tile.first + wid * 32, kj = key0 + (lane & 31);
  const int last = min(tile.first + 127, n - 1), wlast = min(key0 + 31, n - 1);
  const int qbeg = max(tile.first - right, 0) & ~(BK - 1), qend = min(last + left + 1, n);
  const int tiles = query_tiles(a, tile), heads = a.heads / a.kv_heads, parts = parts_of(tiles * heads, split);
  if (sub >= parts) return;
  f32x4* to = parts > 1 ? part + ((size_t)(num * a.kv_heads + kvh) * split.split + sub) * (DP / 4 * 256) : nullptr;  // where this part's sums go
  int from = 0, steps = tiles * heads;  // this part's first step, its steps
  if (parts > 1) {
    from = (int)((long long)steps * sub / parts);
    steps = (int)((long long)steps * (sub + 1) / parts) - from;
  }
  const int h0 = kvh * heads + (parts > 1 ? from / tiles : 0), first = qbeg + (parts > 1 ? from % tiles * BK : 0);
  const float sl2 = a.scale * kLog2e;
  const bool alive = kj < n && (!a.mask || a.mask[tile.row0 + kj] != 0);
  const uint32_t live = (uint32_t)__ballot(alive);  // (both halves of the wave have the same 32 keys)

  constexpr int TB = BK * DP * 2, SB = 2 * TB + 2 * BK * 4, NC = DP / 16, ND = DP / 32;  // Q tile, dO tile, -lse and -delta of the rows
  const uint32_t lds0 = lds_addr(smem);
  Stager<DP> sq(a.q_row, a.dim, lane, wid), sd(a.do_row, a.dim, lane, wid);
  // the tile that is sent for next: its first row, where its Q, dO and statistics are, and from there to the next head's first tile
  int fq = first;
  const uint16_t* qs = a.q + (long long)(tile.row0 + first) * a.q_row + h0 * a.q_head;
  const uint16_t* ds = dctx + (long long)(tile.row0 + first) * a.do_row + h0 * a.do_head;
  const float* st = (wid == 0 ? nlse : ndelta) + (size_t)h0 * a.T + tile.row0 + first;
  const long long qwrap = a.q_head - (long long)tiles * BK * a.q_row, dwrap = a.do_head - (long long)tiles * BK * a.do_row;
  const int swrap = a.T - tiles * BK;
  auto fetch = [&](uint32_t to) {
    const uint64_t rows = bits_below(n - fq);
    const int l = fresh_lane();
    sq.first = sq.first_of(l);
    sd.first = sd.first_of(l);
    sq.all(qs, to + wid * 1024, rows);
    sd.all(ds, to + TB + wid * 1024, rows);
    if (wid < 2) {
      const rsrc_t rs = rsrc_of(st, (uint32_t)min(n - fq, BK) * 4u);
      rsrc_settled(rs);
      dma4(rs, (uint32_t)fresh_lane() * 4u, to + 2 * TB + wid * BK * 4);
    }
    fq += BK;
    qs += sq.ldb * (BK / 2);
    ds += sd.ldb * (BK / 2);
    st += BK;
    if (fq >= qend) {
      fq = qbeg;
      qs += qwrap;
      ds += dwrap;
      st += swrap;
    }
  };
  if (steps) fetch(lds0);

  bf16x8 kf[NC], vf[NC];
  load_frags<DP>(kf, a.k + (long long)(tile.row0 + kj) * a.k_row + kvh * a.k_head, a.dim, alive, half);
  load_frags<DP>(vf, a.v + (long long)(tile.row0 + kj) * a.v_row + kvh * a.v_head, a.dim, alive, half);
  landed(kf);
  landed(vf);
  // (of the 128-wide head's fragments the last three are kept in LDS, each lane its own, and read when they are needed: in registers they are too many)
  constexpr int LENT = DP == 128 ? 3 : 0;
#pragma unroll
  for (int i = 0; i < LENT; ++i) *lds_at<bf16x8>(lds0 + 2 * SB + i * 4096 + tid * 16) = kf[NC - LENT + i];
  f32x16 gk[ND], gv[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) { gk[dt][r] = 0.f; gv[dt][r] = 0.f; }
  Bits<DP> f(lds0, lane);

  int q0 = first, left_ = steps;  // the tile that is worked on, the tiles that are left
  auto work = [&](auto buf_) {
    constexpr int QA = decltype(buf_)::value * SB, DA = QA + TB;
    dma_wait();
    __syncthreads();
    if (--left_ > 0) fetch(lds0 + (decltype(buf_)::value ^ 1) * SB);
    const int at = q0;
    q0 = q0 + BK >= qend ? qbeg : q0 + BK;
    if (live == 0 || at > wlast + left || at + BK <= key0 - right) return;
    const bool edge = live != ~0u || at < wlast - right || at + BK > key0 + left + 1;
    each<2>([&](auto qb_) {
      constexpr int qb = decltype(qb_)::value, Q = QA + qb * 32 * DP * 2, D = DA + qb * 32 * DP * 2;
      // (none of these 32 sees a key of the wave; as in dQ)
      if (DP == 128 && (at + qb * 32 >= qend || at + qb * 32 > wlast + left || at + qb * 32 + 32 <= key0 - right)) return;
      // (fragments are read DEEP - 1 ahead of their products: more do not fit)
      constexpr int DEEP = 3;
      f.forget();
      const uint32_t stat = lds0 + 2 * TB + 16 * (fresh_lane() >> 5);
      f32x16 s, dp;
      bf16x8 x[DEEP], kl[LENT + 1];
      SCHED_FENCE();
#pragma unroll
      for (int c = 0; c < DEEP - 1; ++c) x[c] = f.template row<Q>(c);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        SCHED_FENCE();
        const int u = c + DEEP - 1;
        x[u % DEEP] = u < NC ? f.template row<Q>(u) : f.template row<D>(u - NC);
        const int i = c - (NC - LENT);
        if (i + 1 >= 0 && i + 1 < LENT) kl[i + 1] = *lds_at<const bf16x8>(lds0 + 2 * SB + (i + 1) * 4096 + wid * 1024 + fresh_lane() * 16);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[c % DEEP], i >= 0 ? kl[i] : kf[c], s, 0, 0, 0);
      }
      SCHED_FENCE();
      if (edge) {
        const int l = fresh_lane(), key = key0 + (l & 31), base = at + qb * 32;
        const uint32_t see = (live >> (l & 31)) & 1 ? bits32(key - right - base, min(key + left + 1, n) - base) >> (4 * (l >> 5)) : 0u;
        each<16>([&](auto r_) {
          constexpr int r = decltype(r_)::value;
          s[r] = seen<8 * (r >> 2) + (r & 3)>(see, s[r]);
        });
      }
      SCHED_FENCE();
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {  // dP starts at -delta of its rows
        const f32x4 d4 = *lds_at<const f32x4>(stat + decltype(buf_)::value * SB + BK * 4 + qb * 128 + 32 * rg);
        dp[rg * 4] = d4[0]; dp[rg * 4 + 1] = d4[1]; dp[rg * 4 + 2] = d4[2]; dp[rg * 4 + 3] = d4[3];
      }
      // beside the products of dP: the probabilities, two registers a product
      f32x4 l4;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        SCHED_FENCE();
        const int u = c + DEEP - 1;
        if (u < NC) x[(NC + u) % DEEP] = f.template row<D>(u);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[(NC + c) % DEEP], vf[c], dp, 0, 0, 0);
#pragma unroll
        for (int e = c * 16 / NC; e < (c + 1) * 16 / NC; ++e) {
          if (e % 4 == 0) l4 = *lds_at<const f32x4>(stat + decltype(buf_)::value * SB + qb * 128 + 8 * e);
          s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], sl2, l4[e % 4]));
        }
      }
      SCHED_FENCE();
      bf16x8 pf[2], df[2], z[DEEP];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float p[8], d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = s[j * 8 + e];
          d[e] = s[j * 8 + e] * dp[j * 8 + e];
        }
        pf[j] = as_bf16x8(pack8(p));
        df[j] = as_bf16x8(pack8(d));
        SCHED_FENCE();
      }
      // the steps j of 16 rows: dV's products, then dK's.  fragment k = 2 ND j + ND (dK) + dt
      auto frag = [&](auto k_) {
        constexpr int k = decltype(k_)::value, j = k / (2 * ND), dt = k % ND;
        if constexpr (k % (2 * ND) < ND) return f.template col<D + j * 16 * DP * 2>(dt);
        else return f.template col<Q + j * 16 * DP * 2>(dt);
      };
      each<DEEP - 1>([&](auto k) { z[decltype(k)::value] = frag(k); });
      each<4 * ND>([&](auto k_) {
        constexpr int k = decltype(k_)::value, j = k / (2 * ND), dt = k % ND, u = k + DEEP - 1;
        SCHED_FENCE();
        if constexpr (u < 4 * ND) z[u % DEEP] = frag(std::integral_constant<int, u>{});
        if constexpr (k % (2 * ND) < ND) gv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z[k % DEEP], pf[j], gv[dt], 0, 0, 0);
        else gk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z[k % DEEP], df[j], gk[dt], 0, 0, 0);
      });
      SCHED_FENCE();
    });
  };
  while (left_ > 0) {
    work(std::integral_constant<int, 0>{});
    if (left_ > 0) work(std::integral_constant<int, 1>{});
  }
  if (to) {
    to += tid;
#pragma unroll
    for (int i = 0; i < ND * 8; ++i) {
      const f32x16& g = i < ND * 4 ? gk[i / 4] : gv[i / 4 - ND];
      to[i * 256] = f32x4{g[(i & 3) * 4], g[(i & 3) * 4 + 1], g[(i & 3) * 4 + 2], g[(i & 3) * 4 + 3]};
    }
    return;
  }
  const long long row = tile.row0 + kj;
  store_T<DP>(dk + row * a.dk_row + kvh * a.dk_head, gk, a.scale, a.dim, kj < n, half);
  store_T<DP>(dv + row * a.dv_row + kvh * a.dv_head, gv, 1.0f, a.dim, kj < n, half);
}

// The sums of the parts, in their order.  A thread has the accumulators that the same thread of the parts' workgroups left.
template <int DP>
__global__ __launch_bounds__(256) void attn_gqa_join_kernel(const Args a, const f32x4* __restrict__ part, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv,
                                                            Split split, int order) {
  constexpr int ND = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.kv_heads, num = blockIdx.x / a.kv_heads, heads = a.heads / a.kv_heads;
  const Tile tile = find_tile<128>(a.seq_off, a.B, a.T, num, order, lane);
  if (tile.n == 0) return;
  const int parts = parts_of(query_tiles(a, tile) * heads, split);
  if (parts == 1) return;
  const f32x4* from = part + (size_t)blockIdx.x * split.split * (ND * 8 * 256) + tid;
  const int kj = tile.first + wid * 32 + (lane & 31);
  const long long row = tile.row0 + kj;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    f32x16 g[ND];
#pragma unroll
    for (int i = 0; i < ND * 4; ++i) {
      f32x4 sum = from[(which * ND * 4 + i) * 256];
      for (int s = 1; s < parts; ++s) sum += from[(s * ND * 8 + which * ND * 4 + i) * 256];
#pragma unroll
      for (int e = 0; e < 4; ++e) g[i / 4][(i & 3) * 4 + e] = sum[e];
    }
    if (which == 0) store_T<DP>(dk + row * a.dk_row + kvh * a.dk_head, g, a.scale, a.dim, kj < tile.n, half);
    else store_T<DP>(dv + row * a.dv_row + kvh * a.dv_head, g, 1.0f, a.dim, kj < tile.n, half);
  }
}

// ------------------------------------------------------------------------------------------------ host
constexpr long long kMaxGroups = (1ll << 24) - 1;  // workgroups of 256: a launch counts its work-items in 32 bits
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
  CK_ARG(units <= kMaxGroups, "%s: %d rows in %d sequences of %d heads are too many for one launch (rows / 128 + sequences, times heads: below 2^24)", what, a->T, a->B, a->heads);
  return COCODR_OK;
}

// by work: where tiles have so much of it (sequences of 256 rows and more on average) that the longer search for them does not count, where their work
// differs (no window on both sides), and where a lane each does for the sequences.  Forward and backward, 32 / 8 heads of 128, causal: 4 x 4096 2393 us by
// work, 2690 in the order of the rows; 16 sequences of 1 to 2048 600 and 610.
Order order_of(const Args* a, bool keys) {
  if (a->B > 64 || a->T / a->B < 256 || (a->left >= 0 && a->right >= 0)) return kPlain;
  if (a->left < 0 && a->right < 0) return kLevel;
  return (a->right >= 0) != keys ? kUp : kDown;
}

// Tiles of the dK / dV kernel, and in how many parts it sums a tile's steps.  The chip holds 512 of its workgroups: with fewer tiles than that the
// longest one is all that runs in the end - 16 sequences of 1 to 2048, causal, 32 / 8 heads of 128: 4 x 2048 rows of queries at 2.9 us a step of 64, 373 us of 600.
// As many parts as fit the chip twice (there: two, 205 us and 20 for the join; four, 1888 workgroups, took 543 us for all against 496), and each of more
// steps than what its sums cost, 2 x 128 x D fp32 written and read again.  Backward, us, with parts of more than 48 / 24 / 12 / 8 steps:
//   heads of 128, 32 / 8, causal: 2048 rows 290 / 235 / 191 / 191 (whole: 338), 3 x 2048 440 / 427 / 405 / 394; the 16 sequences with the forward 444 / 448 / 451
//   from 24 on; heads of 64, whose steps are half as long: 4 x 512, 12 heads 34 / 34 / 42 / 37, sequences of 1000, 200 and 50, 16 heads 51 / 51 / 52 / 54
long long units_of(const Args* a) { return ((long long)a->T / 128 + a->B) * a->kv_heads; }
Split split_for(const Args* a) {
  Split s{1, a->dim <= 64 ? 24 : 12};
  const long long steps = ((long long)a->T / 64 + 1) * (a->heads / a->kv_heads);  // of the longest tile, at most
  while (units_of(a) * 2 * s.split <= 1024 && steps > (long long)s.part * 2 * s.split) s.split *= 2;
  return s;
}
size_t stats_floats(const Args* a) { return ((size_t)2 * a->T * a->heads + 3) & ~(size_t)3; }  // (what is behind them starts at a multiple of 16 bytes)
size_t part_floats(const Args* a) { return (size_t)2 * 128 * (a->dim <= 64 ? 64 : 128); }

// the strides between the rows of a single row may be anything, and the kernels' tiles reach as far as 64 strides
Args tidy(const Args* a) {
  Args b = *a;
  if (b.T == 1) b.q_row = b.k_row = b.v_row = b.o_row = b.do_row = b.dq_row = b.dk_row = b.dv_row = 0;
  return b;
}

template <class K> void allow_lds(K kernel, int bytes) { (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); }
constexpr int kv_lds(int DP) { return 4 * BK * DP * 2; }
constexpr int qd_lds(int DP) { return 2 * (2 * BK * DP * 2 + 2 * BK * 4) + (DP == 128 ? 3 * 4096 : 0); }
void lds_limits() {
  static cocodr_lds_once once;
  if (!once.pending()) return;
  allow_lds(attn_gqa_fwd_kernel<64>, kv_lds(64)); allow_lds(attn_gqa_fwd_kernel<128>, kv_lds(128));
  allow_lds(attn_gqa_dq_kernel<64>, kv_lds(64)); allow_lds(attn_gqa_dq_kernel<128>, kv_lds(128));
  allow_lds(attn_gqa_dkv_kernel<64>, qd_lds(64)); allow_lds(attn_gqa_dkv_kernel<128>, qd_lds(128));
  once.done();
}

}  // namespace

extern "C" int cocodr_attn_gqa_fwd(const cocodr_attn_gqa_args* args, uint16_t* ctx, float* lse, int fill, cocodr_stream_t stream) {
  if (int rc = check(args, "attn_gqa_fwd")) return rc;
  const Args b = tidy(args), *a = &b;
  CK_ARG(ctx && lse && aligned16(ctx), "attn_gqa_fwd: ctx and lse must be given, ctx 16-byte aligned");
  CK_ARG(stride_ok(a->o_row, a->o_head, a->T, a->heads) && apart(a->o_row, a->o_head, a->T, a->heads, a->dim), "attn_gqa_fwd: ctx strides must be multiples of 8 and keep its rows apart");
  lds_limits();
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((a->T / 128 + a->B) * a->heads));
  if (a->dim <= 64) hipLaunchKernelGGL(attn_gqa_fwd_kernel<64>, grid, dim3(256), kv_lds(64), st, *a, ctx, lse, order_of(a, false), fill);
  else hipLaunchKernelGGL(attn_gqa_fwd_kernel<128>, grid, dim3(256), kv_lds(128), st, *a, ctx, lse, order_of(a, false), fill);
  CK_LAUNCH("attn_gqa_fwd");
  return COCODR_OK;
}

extern "C" size_t cocodr_attn_gqa_bwd_workspace_floats(const cocodr_attn_gqa_args* a) {
  if (!a || a->T <= 0 || a->B <= 0 || a->kv_heads <= 0 || a->heads < a->kv_heads) return 0;
  const Split s = split_for(a);
  return stats_floats(a) + (s.split > 1 ? (size_t)units_of(a) * s.split * part_floats(a) : 0);
}

extern "C" int cocodr_attn_gqa_bwd(const cocodr_attn_gqa_args* args, const uint16_t* ctx, const uint16_t* dctx, const float* lse, uint16_t* dq,
                                   uint16_t* dk, uint16_t* dv, int fill, float* workspace, size_t workspace_floats, cocodr_stream_t stream) {
  if (int rc = check(args, "attn_gqa_bwd")) return rc;
  const Args b = tidy(args), *a = &b;
  CK_ARG(ctx && dctx && lse && dq && dk && dv, "attn_gqa_bwd: null pointer");
  CK_ARG(aligned16(ctx) && aligned16(dctx) && aligned16(dq) && aligned16(dk) && aligned16(dv), "attn_gqa_bwd: tensors must be 16-byte aligned");
  CK_ARG(stride_ok(a->o_row, a->o_head, a->T, a->heads) && stride_ok(a->do_row, a->do_head, a->T, a->heads), "attn_gqa_bwd: strides must be multiples of 8 elements, rows less than 2^23 apart");
  CK_ARG(stride_ok(a->dq_row, a->dq_head, a->T, a->heads) && apart(a->dq_row, a->dq_head, a->T, a->heads, a->dim) && stride_ok(a->dk_row, a->dk_head, a->T, a->kv_heads) &&
             apart(a->dk_row, a->dk_head, a->T, a->kv_heads, a->dim) && stride_ok(a->dv_row, a->dv_head, a->T, a->kv_heads) && apart(a->dv_row, a->dv_head, a->T, a->kv_heads, a->dim),
         "attn_gqa_bwd: gradient strides must be multiples of 8 and keep the rows apart");
  CK_ARG(aligned16(workspace), "attn_gqa_bwd: the workspace must be 16-byte aligned");
  if (!workspace || workspace_floats < cocodr_attn_gqa_bwd_workspace_floats(a)) {
    cocodr_set_error("attn_gqa_bwd: workspace of %zu floats is too small", workspace_floats);
    return COCODR_ERR_WORKSPACE;
  }
  lds_limits();
  hipStream_t st = (hipStream_t)stream;
  float *ndelta = workspace, *nlse = workspace + (size_t)a->T * a->heads;
  f32x4* part = reinterpret_cast<f32x4*>(workspace + stats_floats(a));
  const Split split = split_for(a);
  const Order rows = order_of(a, false), keys = order_of(a, true);
  const dim3 gq((unsigned)((a->T / 128 + a->B) * a->heads)), gk((unsigned)(units_of(a) * split.split)), gj((unsigned)units_of(a));
  if (a->dim <= 64) {
    hipLaunchKernelGGL(attn_gqa_dq_kernel<64>, gq, dim3(256), kv_lds(64), st, *a, ctx, dctx, lse, ndelta, nlse, dq, rows, fill);
    hipLaunchKernelGGL(attn_gqa_dkv_kernel<64>, gk, dim3(256), qd_lds(64), st, *a, dctx, ndelta, nlse, dk, dv, part, split, keys, fill);
    if (split.split > 1) hipLaunchKernelGGL(attn_gqa_join_kernel<64>, gj, dim3(256), 0, st, *a, part, dk, dv, split, keys);
  } else {
    hipLaunchKernelGGL(attn_gqa_dq_kernel<128>, gq, dim3(256), kv_lds(128), st, *a, ctx, dctx, lse, ndelta, nlse, dq, rows, fill);
    hipLaunchKernelGGL(attn_gqa_dkv_kernel<128>, gk, dim3(256), qd_lds(128), st, *a, dctx, ndelta, nlse, dk, dv, part, split, keys, fill);
    if (split.split > 1) hipLaunchKernelGGL(attn_gqa_join_kernel<128>, gj, dim3(256), 0, st, *a, part, dk, dv, split, keys);
  }
  CK_LAUNCH("attn_gqa_bwd");
  return COCODR_OK;
}
