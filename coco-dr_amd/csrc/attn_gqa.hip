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
#include "common.h"
#include "prof.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;  // where a running maximum starts: finite, so that a row without any key gives exp2(-inf - kLow) = 0 and no NaN
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

// BK rows of one head into a tile by LDS DMA: a wave's instruction writes 1 KiB lane-linear, so the permutation goes into the source
// addresses.  Rows whose bit of `rows` is 0 (behind the sequence, masked out) and columns >= D are addressed behind the descriptor's
// end and arrive as zeros: whatever stands there in memory, NaN too, is not read.  src: the tile's first row (the descriptor reaches
// over one tile only, so its 32-bit offsets do for any buffer).
template <int DP> __device__ __forceinline__ void stage(char* dst, const uint16_t* src, long long ld, int D, uint64_t rows, int lane, int wid) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int CH = DP / 8, RP = 64 / CH;  // chunks of a row, rows of a piece
  const uint32_t ldb = (uint32_t)ld * 2u;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, (uint32_t)(BK - 1) * ldb + (uint32_t)D * 2u, 0x00020000);
#pragma unroll
  for (int i = 0; i < BK / RP / 4; ++i) {
    const int p = wid + i * 4;
    const int row = p * RP + lane / CH, ch = (lane & (CH - 1)) ^ swz<DP>(row);
    const uint32_t off = ((rows >> row) & 1) && ch * 8 < D ? (uint32_t)row * ldb + (uint32_t)ch * 16u : 0x80000000u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_PTR(void))(dst + p * 1024), 16, off, 0, 0, 0);
  }
#endif
}
// one row's operand fragments straight from memory (the operand that a wave keeps): zeros where `ok` is false and behind column D
template <int DP> __device__ __forceinline__ void load_frags(bf16x8 (&f)[DP / 16], const uint16_t* row, int D, bool ok, int half) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int col = (2 * s + half) * 8;
    f[s] = as_bf16x8(ok && col < D ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0u, 0u, 0u, 0u));
  }
}

__device__ __forceinline__ bf16x8 pack_acc(const float* p, int j) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = p[j * 8 + e];
  return as_bf16x8(pack8(t));
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
// A workgroup has 128 query rows of one head, each of its four waves 32 of them; K and V pass through LDS in tiles of 64 keys, two
// tiles each, so that a tile is on its way while the one before is worked on.
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_gqa_fwd_kernel(const Args a, uint16_t* __restrict__ ctx, float* __restrict__ lse, int fill) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (fill) {
    const Gaps gap(a.seq_off, a.B, a.T);
    for (long long i = blockIdx.x; i < (long long)gap.count * a.heads; i += gridDim.x) {
      const int row = gap.row((int)(i / a.heads)), h = (int)(i % a.heads);
      if (tid * 4 < a.dim) *reinterpret_cast<uint2*>(ctx + row * a.o_row + h * a.o_head + tid * 4) = make_uint2(0u, 0u);
      if (tid == 0) lse[(size_t)h * a.T + row] = -INFINITY;
    }
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

  bf16x8 qf[DP / 16];
  load_frags<DP>(qf, a.q + (long long)(tile.row0 + qi) * a.q_row + h * a.q_head, a.dim, qi < n, half);
  f32x16 o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = kLow, l = 0.f;

  constexpr int TB = BK * DP * 2;  // bytes of a tile
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  if (kbeg < kend) {
    stage<DP>(smem, kb_ + kbeg * a.k_row, a.k_row, a.dim, word, lane, wid);
    stage<DP>(smem + TB, vb_ + kbeg * a.v_row, a.v_row, a.dim, word, lane, wid);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
    const char* Kt = smem + buf * 2 * TB;
    const char* Vt = Kt + TB;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint64_t next = key_word(a.mask, loaded, n, k0 + BK);
    if (k0 + BK < kend) {
      char* to = smem + (buf ^ 1) * 2 * TB;
      stage<DP>(to, kb_ + (long long)(k0 + BK) * a.k_row, a.k_row, a.dim, next, lane, wid);
      stage<DP>(to + TB, vb_ + (long long)(k0 + BK) * a.v_row, a.v_row, a.dim, next, lane, wid);
      loaded = key_word_load(a.mask, tile.row0, n, k0 + 2 * BK, lane);
    }
    const uint64_t now = word;
    word = next;
    if (q0 >= n || k0 > wlast + right || k0 + BK <= q0 - left || now == 0) continue;  // this wave's rows see nothing of the tile
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows<DP>(Kt, kb * 32, c, lane), qf[c], s[kb], 0, 0, 0);
    }
    if (now != ~0ull || k0 < wlast - left || k0 + BK > q0 + right + 1) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int base = k0 + kb * 32;
        const uint32_t see = (bits32(qi - left - base, qi + right + 1 - base) & (uint32_t)(now >> (kb * 32))) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = (see >> (8 * (r >> 2) + (r & 3))) & 1 ? s[kb][r] : -INFINITY;
      }
    }
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
    top = fmaxf(top, __shfl_xor(top, 32, 64)) * sl2;
    if (__any(top > m + 8.0f)) {  // (a maximum that grows by less than 2^8 is left: sums of up to 2^8-fold terms are as exact in fp32)
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], sl2, -m));
        l += p[r];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x8 pf = pack_acc(p, j);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols<DP>(Vt, kb * 32 + j * 16, dt, lane), pf, o[dt], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (qi < n && lane < 32) lse[(size_t)h * a.T + tile.row0 + qi] = l > 0.f ? (m + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
  store_T<DP>(ctx + (long long)(tile.row0 + qi) * a.o_row + h * a.o_head, o, l > 0.f || l != l ? 1.0f / l : 0.f, a.dim, qi < n, half);
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
  const float nl = qi < n ? -lse[at] * kLog2e : 0.f;
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
    nd += __shfl_xor(nd, 32, 64);
  }
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
  int loaded = key_word_load(a.mask, tile.row0, n, kbeg, lane);
  uint64_t word = key_word(a.mask, loaded, n, kbeg);
  loaded = key_word_load(a.mask, tile.row0, n, kbeg + BK, lane);
  if (kbeg < kend) {
    stage<DP>(smem, kb_ + kbeg * a.k_row, a.k_row, a.dim, word, lane, wid);
    stage<DP>(smem + TB, vb_ + kbeg * a.v_row, a.v_row, a.dim, word, lane, wid);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
    const char* Kt = smem + buf * 2 * TB;
    const char* Vt = Kt + TB;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint64_t next = key_word(a.mask, loaded, n, k0 + BK);
    if (k0 + BK < kend) {
      char* to = smem + (buf ^ 1) * 2 * TB;
      stage<DP>(to, kb_ + (long long)(k0 + BK) * a.k_row, a.k_row, a.dim, next, lane, wid);
      stage<DP>(to + TB, vb_ + (long long)(k0 + BK) * a.v_row, a.v_row, a.dim, next, lane, wid);
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
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) { gk[dt][r] = 0.f; gv[dt][r] = 0.f; }

  constexpr int TB = BK * DP * 2, SB = 2 * TB + 2 * BK * 4;  // Q tile, dO tile, -lse and -delta of the rows
  const int tiles = qend > qbeg ? (qend - qbeg + BK - 1) / BK : 0, steps = tiles * G;
  auto fetch = [&](int i, char* to) {
    const int h = kvh * G + i / tiles, q0 = qbeg + (i % tiles) * BK;
    const uint64_t rows = bits_below(n - q0);
    stage<DP>(to, a.q + (long long)(tile.row0 + q0) * a.q_row + h * a.q_head, a.q_row, a.dim, rows, lane, wid);
    stage<DP>(to + TB, dctx + (long long)(tile.row0 + q0) * a.do_row + h * a.do_head, a.do_row, a.dim, rows, lane, wid);
#if defined(__HIP_DEVICE_COMPILE__)
    if (wid < 2) {
      const float* src = (wid == 0 ? nlse : ndelta) + (size_t)h * a.T + tile.row0 + q0;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, (uint32_t)min(n - q0, BK) * 4u, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_PTR(void))(to + 2 * TB + wid * BK * 4), 4, (uint32_t)lane * 4u, 0, 0, 0);
    }
#endif
  };
  if (steps) fetch(0, smem);
  for (int i = 0; i < steps; ++i) {
    const char* Qt = smem + (i & 1) * SB;
    const char* Dt = Qt + TB;
    const float* nl = reinterpret_cast<const float*>(Qt + 2 * TB);
    const float* nd = nl + BK;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (i + 1 < steps) fetch(i + 1, smem + ((i + 1) & 1) * SB);
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

template <class K> void allow_lds(K kernel, int bytes) { (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); }
constexpr int kv_lds(int DP) { return 4 * BK * DP * 2; }
constexpr int qd_lds(int DP) { return 2 * (2 * BK * DP * 2 + 2 * BK * 4); }
void lds_limits() {
  static cocodr_lds_once once;
  if (!once.pending()) return;
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
  if (a->dim <= 64) hipLaunchKernelGGL(attn_gqa_fwd_kernel<64>, grid, dim3(256), kv_lds(64), st, *a, ctx, lse, fill);
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
