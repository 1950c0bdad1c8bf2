// Embedding lookup with scaling, and its gradient by sorted tokens.
//   out_t = scale E[id_t]          dE_v = scale sum over t with id_t = v, in the order of t, of dout_t
// An id outside [0, vocab) is a padding row: zeros out, no gradient.  Both are bound by memory: the looked-up rows in and out; dout in and
// the dense gradient (the whole table, zeros included) out.
//
// The gradient adds no floats atomically: its sums run in the order of the tokens, so the same inputs give the same bits.  The tokens of each id are
// brought together by counting:
//   rank    a token's number among those of its id, and how many there are (integer atomics: their order is arbitrary)
//   alloc   every id that occurs takes a stretch of the position list; ids with more than kFew tokens go to a list of their own
//   place   positions into the stretches
//   sum     a wave per table row: the row's positions are put in order (they are few: every lane counts how many are smaller than its own)
//           and the rows of dout added; an id with many tokens is worked on by whole workgroups, one for every 512 columns and window of
//           positions, which mark the positions in a bitmap in LDS and read them back in order
//   join    the windows' sums of those ids, in order
#include <algorithm>
#include "common.h"

namespace {

constexpr int kFew = 64;          // tokens of an id that one wave orders by itself: one per lane
constexpr int kWindows = 8;       // parts that the tokens of a frequent id are split into, by position
constexpr int kWindowMin = 4096;  // positions of a part at least
constexpr int kMap = 1 << 16;     // positions that the bitmap holds at a time (8 KiB)
constexpr int kBatch = 1024;      // ordered positions at a time
constexpr int kSlice = 512;       // columns: 64 lanes x 8

struct Ids {
  const void* p;
  int wide;  // 64-bit
  __device__ __forceinline__ long long at(int i) const { return wide ? ((const long long*)p)[i] : (long long)((const int32_t*)p)[i]; }
};

template <bool F32> __device__ __forceinline__ void load8(const void* base, size_t i, float (&v)[8]) {
  if constexpr (F32) {
    const float4* q = reinterpret_cast<const float4*>((const float*)base + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else unpack8(*reinterpret_cast<const uint4*>((const uint16_t*)base + i), v);
}
template <bool F32> __device__ __forceinline__ void store8(void* base, size_t i, const float (&v)[8]) {
  if constexpr (F32) {
    float4* q = reinterpret_cast<float4*>((float*)base + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else *reinterpret_cast<uint4*>((uint16_t*)base + i) = pack8(v);
}

// ------------------------------------------------------------------------------------------------ lookup
// a workgroup has `per` rows; a thread 8 columns at a time
template <bool TF32, bool OF32>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const Ids ids, const void* __restrict__ table, void* __restrict__ out, int n, int H, int vocab,
                                                        float scale, int per) {
  const unsigned nch = (unsigned)H >> 3;
  const int row0 = blockIdx.x * per, rows = min(per, n - row0);
  for (unsigned i = threadIdx.x; i < (unsigned)rows * nch; i += 256) {
    const unsigned r = i / nch, c = i - r * nch;
    const long long id = ids.at(row0 + (int)r);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (id >= 0 && id < vocab) {
      load8<TF32>(table, (size_t)id * H + c * 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= scale;
    }
    store8<OF32>(out, (size_t)(row0 + (int)r) * H + c * 8, v);
  }
}

// ------------------------------------------------------------------------------------------------ gradient
// ints of the workspace: count [vocab], begin [vocab], rank [n], pos [n], many [n / kFew + 1], cursor [2] (positions taken, frequent ids)
struct Plan {
  int *count, *begin, *rank, *pos, *many, *cursor;
  float* parts;  // [frequent ids][windows][H]
  int windows, window;
};
size_t round4(size_t x) { return (x + 3) & ~(size_t)3; }
int windows_of(int n) { return std::max(1, std::min(kWindows, n / kWindowMin)); }
size_t plan_of(int* ws, int n, int H, int vocab, Plan& p) {
  size_t at = 0;
  auto take = [&](size_t ints) { int* q = ws + at; at += round4(ints); return q; };
  p.cursor = take(2);
  p.count = take(vocab);  // (behind the cursors: one fill clears both)
  p.begin = take(vocab);
  p.rank = take(n);
  p.pos = take(n);
  p.many = take(n / kFew + 1);
  p.windows = windows_of(n);
  p.window = (n + p.windows - 1) / p.windows;
  p.parts = (float*)(ws + at);
  if (p.windows > 1) at += round4((size_t)(n / (kFew + 1) + 1) * p.windows * H);
  return at;
}

__global__ __launch_bounds__(256) void embed_clear_kernel(int4* p, size_t n4) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (size_t)gridDim.x * 256) p[i] = make_int4(0, 0, 0, 0);
}

// Lanes of one id take their numbers with a single atomic: a batch of one repeated token would otherwise wait for n atomics on one address.
__global__ __launch_bounds__(256) void embed_rank_kernel(const Ids ids, int n, int vocab, int* __restrict__ count, int* __restrict__ rank) {
  const int i = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 63;
  long long id = i < n ? ids.at(i) : -1;
  const bool ok = id >= 0 && id < vocab;
  int mine = -1;
  uint64_t left = __ballot(ok);
  while (left) {
    const int lead = (int)__builtin_ctzll(left);
    const int v = __builtin_amdgcn_readlane((int)id, lead);
    const uint64_t same = __ballot(ok && (int)id == v) & left;
    if (ok && (int)id == v) {
      int base = 0;
      if (lane == lead) base = atomicAdd(count + v, (int)__popcll(same));
      base = __builtin_amdgcn_readlane(base, lead);
      mine = base + (int)__popcll(same & ((1ull << lane) - 1ull));
    }
    left &= ~same;
  }
  if (i < n) rank[i] = mine;
}

__global__ __launch_bounds__(1024) void embed_alloc_kernel(const int* __restrict__ count, int* __restrict__ begin, int* __restrict__ many, int* cursor, int vocab) {
  __shared__ int part[17];
  const int v = blockIdx.x * 1024 + threadIdx.x, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int c = v < vocab ? count[v] : 0;
  int sum = c;  // inclusive over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  if (lane == 63) part[wid] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    int run = 0;
    for (int w = 0; w < 16; ++w) {
      const int x = part[w];
      part[w] = run;
      run += x;
    }
    part[16] = run ? atomicAdd(cursor, run) : 0;
  }
  __syncthreads();
  if (v < vocab) begin[v] = part[16] + part[wid] + sum - c;
  if (c > kFew) many[atomicAdd(cursor + 1, 1)] = v;
}

__global__ __launch_bounds__(256) void embed_place_kernel(const Ids ids, int n, const int* __restrict__ begin, const int* __restrict__ rank, int* __restrict__ pos) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int r = rank[i];
  if (r >= 0) pos[begin[(int)ids.at(i)] + r] = i;
}

__device__ __forceinline__ void put_row(float* out, size_t at, const float (&acc)[8], float scale, int add) {
  float v[8];
  if (add) {
    load8<true>(out, at, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf(acc[e], scale, v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = acc[e] * scale;
  }
  store8<true>(out, at, v);
}

// one wave, one table row of at most kFew tokens
template <bool F32>
__device__ void sum_few(const void* dout, float* out, int v, int c, const int* pos, int H, float scale, int add, int lane) {
  if (c == 0 && add) return;
  int sorted = 0;
  if (c > 0) {
    const int mine = lane < c ? pos[lane] : INT32_MAX;
    int smaller = 0;
    for (int j = 0; j < c; ++j) smaller += __builtin_amdgcn_readlane(mine, j) < mine;
    // lanes without a position go behind those with one, each to a lane of its own
    sorted = __builtin_amdgcn_ds_permute((lane < c ? smaller : lane) * 4, mine);
  }
  // (every lane takes every turn, those behind the last column on column 0: a lane that is read from has to be active)
  for (int col0 = 0; col0 < H; col0 += kSlice) {
    const int col = col0 + lane * 8, from = col < H ? col : 0;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int j = 0;
    for (; j + 4 <= c; j += 4) {
      float x[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) load8<F32>(dout, (size_t)__builtin_amdgcn_readlane(sorted, j + u) * H + from, x[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += x[u][e];
    }
    for (; j < c; ++j) {
      float x[8];
      load8<F32>(dout, (size_t)__builtin_amdgcn_readlane(sorted, j) * H + from, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += x[e];
    }
    if (col < H) put_row(out, (size_t)v * H + col, acc, scale, add);
  }
}

// one workgroup: the tokens of id v at positions [from, to), columns col0 .. col0 + 511.  Wave w adds the ordered positions j with
// (j >> 3) % 4 = w; the four sums are joined in the order of the waves.
template <bool F32>
__device__ void sum_many(const void* dout, float* dst, size_t dst_at, int c, const int* pos, int from, int to, int H, int col0, float scale, int add,
                         uint32_t* map, int* list, float* joined, int* counts) {
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int col = col0 + lane * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int base = from; base < to; base += kMap) {
    const int words = (min(kMap, to - base) + 31) >> 5;
    for (int i = tid; i < words; i += 256) map[i] = 0u;
    __syncthreads();
    for (int i = tid; i < c; i += 256) {
      const int p = pos[i] - base;
      if (p >= 0 && p < kMap && p + base < to) atomicOr(map + (p >> 5), 1u << (p & 31));
    }
    __syncthreads();
    // a stretch of words per thread, its positions behind those of the threads before
    const int per = (words + 255) >> 8, w0 = tid * per, w1 = min(w0 + per, words);
    int have = 0;
    for (int i = w0; i < w1; ++i) have += __popc(map[i]);
    int incl = have;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(incl, d, 64);
      if (lane >= d) incl += up;
    }
    if (lane == 63) counts[wid] = incl;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < 4; ++w) {
      if (w < wid) before += counts[w];
      total += counts[w];
    }
    const int first = before + incl - have;
    for (int b0 = 0; b0 < total; b0 += kBatch) {
      __syncthreads();  // (the list's readers are done, and so are those of counts)
      int at = first;
      if (at + have > b0 && at < b0 + kBatch)
        for (int i = w0; i < w1; ++i)
          for (uint32_t m = map[i]; m; m &= m - 1, ++at)
            if (at >= b0 && at < b0 + kBatch) list[at - b0] = base + i * 32 + __builtin_ctz(m);
      __syncthreads();
      const int got = min(kBatch, total - b0);
      if (col < H)
        for (int j0 = wid * 8; j0 < got; j0 += 32) {
          float x[8][8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const bool is = j0 + u < got;
            load8<F32>(dout, (size_t)list[is ? j0 + u : j0] * H + col, x[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] = is ? x[u][e] : 0.f;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += x[u][e];
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) joined[(wid * 8 + e) * 64 + lane] = acc[e];
  __syncthreads();
  if (wid == 0 && col < H) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = ((joined[e * 64 + lane] + joined[(8 + e) * 64 + lane]) + joined[(16 + e) * 64 + lane]) + joined[(24 + e) * 64 + lane];
    put_row(dst, dst_at + col, acc, scale, add);
  }
  __syncthreads();
}

template <bool F32>
__global__ __launch_bounds__(256) void embed_sum_kernel(const void* __restrict__ dout, float* __restrict__ out, const Plan p, int n, int H, int vocab,
                                                        float scale, int add, int blocks_many) {
  __shared__ uint32_t map[kMap / 32];
  __shared__ int list[kBatch];
  __shared__ float joined[32 * 64];
  __shared__ int counts[4];
  if ((int)blockIdx.x < blocks_many) {  // the frequent ids first: their workgroups take longest
    const int slices = (H + kSlice - 1) / kSlice;
    const long long tasks = (long long)p.cursor[1] * slices * p.windows;
    for (long long t = blockIdx.x; t < tasks; t += blocks_many) {
      const int col0 = (int)(t % slices) * kSlice, w = (int)(t / slices % p.windows), k = (int)(t / slices / p.windows);
      const int v = p.many[k];
      const int from = w * p.window, to = min(from + p.window, n);
      if (p.windows > 1) sum_many<F32>(dout, p.parts, ((size_t)k * p.windows + w) * H, p.count[v], p.pos + p.begin[v], from, to, H, col0, 1.0f, 0, map, list, joined, counts);
      else sum_many<F32>(dout, out, (size_t)v * H, p.count[v], p.pos + p.begin[v], from, to, H, col0, scale, add, map, list, joined, counts);
    }
    return;
  }
  const int v = ((int)blockIdx.x - blocks_many) * 4 + (threadIdx.x >> 6);
  if (v >= vocab) return;
  const int c = __builtin_amdgcn_readfirstlane(p.count[v]);
  if (c <= kFew) sum_few<F32>(dout, out, v, c, p.pos + __builtin_amdgcn_readfirstlane(p.begin[v]), H, scale, add, threadIdx.x & 63);
}

__global__ __launch_bounds__(256) void embed_join_kernel(float* __restrict__ out, const Plan p, int H, float scale, int add) {
  const int nch = H >> 3;
  for (int k = blockIdx.x; k < p.cursor[1]; k += gridDim.x)
    for (int c = threadIdx.x; c < nch; c += 256) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < p.windows; ++w) {
        float x[8];
        load8<true>(p.parts, ((size_t)k * p.windows + w) * H + c * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += x[e];
      }
      put_row(out, (size_t)p.many[k] * H + c * 8, acc, scale, add);
    }
}

int check(const char* what, const void* ids, const void* a, const void* b, int n, int H, int vocab, float scale) {
  CK_ARG(n >= 0 && n < (1 << 30) && vocab > 0 && vocab < (1 << 30), "%s: n=%d rows, vocab=%d: below 2^30, vocab at least 1", what, n, vocab);
  CK_ARG(H > 0 && H % 8 == 0 && H <= (1 << 20), "%s: width %d must be a multiple of 8 up to 2^20", what, H);
  CK_ARG(scale - scale == 0.f, "%s: scale must be finite", what);
  CK_ARG((n == 0 || (ids && a)) && b, "%s: null pointer", what);
  CK_ARG(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0, "%s: tensors must be 16-byte aligned", what);
  return COCODR_OK;
}

}  // namespace

extern "C" int cocodr_embed_fwd(const void* ids, int ids_i64, const void* table, int table_f32, void* out, int out_f32, int n, int H, int vocab, float scale,
                                cocodr_stream_t stream) {
  if (n == 0) return COCODR_OK;
  if (int rc = check("embed_fwd", ids, table, out, n, H, vocab, scale)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int per = std::max(1, 2048 / (H / 8));
  const dim3 grid((unsigned)((n + per - 1) / per));
  const Ids d{ids, ids_i64};
  if (table_f32) {
    if (out_f32) hipLaunchKernelGGL((embed_fwd_kernel<true, true>), grid, dim3(256), 0, st, d, table, out, n, H, vocab, scale, per);
    else hipLaunchKernelGGL((embed_fwd_kernel<true, false>), grid, dim3(256), 0, st, d, table, out, n, H, vocab, scale, per);
  } else {
    if (out_f32) hipLaunchKernelGGL((embed_fwd_kernel<false, true>), grid, dim3(256), 0, st, d, table, out, n, H, vocab, scale, per);
    else hipLaunchKernelGGL((embed_fwd_kernel<false, false>), grid, dim3(256), 0, st, d, table, out, n, H, vocab, scale, per);
  }
  CK_LAUNCH("embed_fwd");
  return COCODR_OK;
}

extern "C" size_t cocodr_embed_bwd_workspace_bytes(int n, int H, int vocab) {
  if (n < 0 || H <= 0 || vocab <= 0) return 0;
  Plan p;
  return plan_of(nullptr, n, H, vocab, p) * sizeof(int);
}

extern "C" int cocodr_embed_bwd(const void* dout, int dout_f32, const void* ids, int ids_i64, float* dtable, int n, int H, int vocab, float scale, int accumulate,
                                void* workspace, size_t workspace_bytes, cocodr_stream_t stream) {
  if (int rc = check("embed_bwd", ids, dout, dtable, n, H, vocab, scale)) return rc;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < cocodr_embed_bwd_workspace_bytes(n, H, vocab)) {
    cocodr_set_error("embed_bwd: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
    return COCODR_ERR_WORKSPACE;
  }
  if (n == 0 && accumulate) return COCODR_OK;
  hipStream_t st = (hipStream_t)stream;
  Plan p;
  plan_of((int*)workspace, n, H, vocab, p);
  const Ids d{ids, ids_i64};
  const size_t clear4 = (round4(2) + round4(vocab)) / 4;
  hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)std::min<size_t>((clear4 + 255) / 256, 1024)), dim3(256), 0, st, (int4*)p.cursor, clear4);
  if (n > 0) {
    hipLaunchKernelGGL(embed_rank_kernel, dim3((n + 255) / 256), dim3(256), 0, st, d, n, vocab, p.count, p.rank);
    hipLaunchKernelGGL(embed_alloc_kernel, dim3((vocab + 1023) / 1024), dim3(1024), 0, st, p.count, p.begin, p.many, p.cursor, vocab);
    hipLaunchKernelGGL(embed_place_kernel, dim3((n + 255) / 256), dim3(256), 0, st, d, n, p.begin, p.rank, p.pos);
  }
  CK_LAUNCH("embed_bwd(order)");
  const int blocks_many = n > kFew ? (int)std::min<long long>(1024, (long long)(n / (kFew + 1)) * ((H + kSlice - 1) / kSlice) * p.windows) : 0;
  const dim3 grid((unsigned)(blocks_many + (vocab + 3) / 4));
  if (dout_f32) hipLaunchKernelGGL(embed_sum_kernel<true>, grid, dim3(256), 0, st, dout, dtable, p, n, H, vocab, scale, accumulate, blocks_many);
  else hipLaunchKernelGGL(embed_sum_kernel<false>, grid, dim3(256), 0, st, dout, dtable, p, n, H, vocab, scale, accumulate, blocks_many);
  if (p.windows > 1) hipLaunchKernelGGL(embed_join_kernel, dim3(std::min(1024, n / (kFew + 1))), dim3(256), 0, st, dtable, p, H, scale, accumulate);
  CK_LAUNCH("embed_bwd");
  return COCODR_OK;
}
