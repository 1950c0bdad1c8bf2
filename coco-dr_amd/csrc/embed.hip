// Embedding lookup with scaling, and its gradient by sorted tokens.
//   out_t = scale E[id_t]          dE_v = scale sum over t with id_t = v, in the order of t, of dout_t
// An id outside [0, vocab) is a padding row: zeros out, no gradient.  Both are bound by memory: the looked-up rows in and out; dout in and
// the dense gradient (the whole table, zeros included) out.
//
// The gradient adds no floats atomically, so the same inputs give the same bits: an id of up to kFew tokens is added up in their order, one with more
// in a fixed tree that follows from their number and positions and, above kMany, from n.  The tokens of each id are brought together by counting:
//   rank    a token's number among those of its id, and how many there are (integer atomics: their order is arbitrary)
//   alloc   every id that occurs takes a stretch of the position list and goes, by the number of its tokens, to the rows that waves work on (up to
//           kFew), to the tasks of whole workgroups (up to kMany) or to the list of those that several workgroups share
//   place   positions into the stretches
//   sum     a wave per such row and 512 columns: its positions are put in order (they are few: every lane counts how many are smaller than its own)
//           and the rows of dout added; a task's workgroup marks the positions of its id in a bitmap in LDS, reads them back in order and adds a
//           slice of the columns, the narrower the more tokens there are, as its lanes that the slice does not need take further rows at the same
//           time; an id with more than kMany tokens has slices of 64 columns and kWindows windows of positions
//   join    the windows' sums of those last ids, in order
#include <algorithm>
#include "common.h"

namespace {

constexpr int kFew = 16;          // tokens of an id that one wave adds by itself, four at a time
// Tokens of an id that one workgroup a slice goes through (128 at a time).  More of them need the join, a launch of its own for every batch that could
// hold such an id: 8192 tokens of text, 30522 x 768, 35 us, 36.6 with a limit of 2048; one id 8192 times 90 us and 44.  32768 tokens of one id 90 us, 488
// with a limit of 32768.
constexpr int kMany = 8192;
constexpr int kWindows = 8;       // windows of positions above that
constexpr int kTaskers = 1024;    // workgroups that go through the tasks
constexpr int kRowers = 4096;     // ... through the rows
constexpr int kFillers = 1024;    // workgroups that clear, beside a launch's own
constexpr int kMap = 1 << 16;     // positions that the bitmap holds at a time (8 KiB)
constexpr int kBatch = 1024;      // ordered positions at a time
constexpr int kWide = 512;        // columns of a wave: 64 lanes x 8
constexpr int kLeast = 8;         // lanes of the narrowest slice: 64 columns, 32 rows at a time
constexpr int kGroups = 1 << 23;  // workgroups of a lookup: 256 work-items each, fewer than 2^32 in all

struct Ids {
  const void* p;
  int wide;  // 64-bit
  __device__ __forceinline__ long long at(int i) const { return wide ? ((const long long*)p)[i] : (long long)((const int32_t*)p)[i]; }
};

template <bool F32> __device__ __forceinline__ float4 load4(const void* base, size_t i) {
  if constexpr (F32) return *reinterpret_cast<const float4*>((const float*)base + i);
  float v[4];
  unpack4(*reinterpret_cast<const uint2*>((const uint16_t*)base + i), v);
  return make_float4(v[0], v[1], v[2], v[3]);
}
template <bool F32> __device__ __forceinline__ void store4(void* base, size_t i, const float4& v) {
  if constexpr (F32) *reinterpret_cast<float4*>((float*)base + i) = v;
  else *reinterpret_cast<uint2*>((uint16_t*)base + i) = make_uint2(pack2bf(v.x, v.y), pack2bf(v.z, v.w));
}
template <bool F32> __device__ __forceinline__ void load8(const void* base, size_t i, float (&v)[8]) {
  if constexpr (F32) {
    const float4* q = reinterpret_cast<const float4*>((const float*)base + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else unpack8(*reinterpret_cast<const uint4*>((const uint16_t*)base + i), v);
}
// ------------------------------------------------------------------------------------------------ lookup
// a workgroup has `per` rows; a thread 4 columns at a time
template <bool TF32, bool OF32>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const Ids ids, const void* __restrict__ table, void* __restrict__ out, int n, int H, int vocab,
                                                        float scale, int per) {
  const unsigned nch = (unsigned)H >> 2;
  const int row0 = blockIdx.x * per, rows = min(per, n - row0);
  for (unsigned i = threadIdx.x; i < (unsigned)rows * nch; i += 256) {
    const unsigned r = i / nch, c = i - r * nch;
    const long long id = ids.at(row0 + (int)r);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (id >= 0 && id < vocab) {
      v = load4<TF32>(table, (size_t)id * H + c * 4);
      v.x *= scale; v.y *= scale; v.z *= scale; v.w *= scale;
    }
    store4<OF32>(out, (size_t)(row0 + (int)r) * H + c * 4, v);
  }
}

// ------------------------------------------------------------------------------------------------ gradient
// lanes that share a row of an id with c tokens: a workgroup's groups of lanes have about 16 rows each
__host__ __device__ __forceinline__ int slice_lanes(int c) {
  int lanes = 256;
  while (lanes > kLeast && c > 16 * (256 / lanes)) lanes >>= 1;
  return lanes;
}
// ints of the workspace: cursor (positions taken, rows, tasks, ids with more than kMany tokens) and count [vocab], cleared at first; begin [vocab],
// rank [n], pos [n], the rows, the tasks - an id with c tokens has ceil(H / (8 lanes)) of them, and 256 / lanes < c / 8: together less than
// n H / 16384 + the number of such ids -, the list of the ids with more than kMany, the windows' sums
struct Plan {
  int *cursor, *count, *begin, *rank, *pos, *most;
  int4 *row, *task;  // (id, tokens, first position in pos, tasks: first column / 8 << 4 | log2 of the slice's lanes)
  float* parts;  // [ids with more than kMany tokens][kWindows][H]
};
size_t round4(size_t x) { return (x + 3) & ~(size_t)3; }
// With fewer tokens than table rows most rows stay zero, and the ordering's launches clear the table as they go; with more tokens nearly every row
// would be written twice, and the rows without tokens are rows of the sum.
bool clears_early(int n, int vocab) { return n <= vocab; }
int rows_at_most(int n, int vocab) { return clears_early(n, vocab) ? n : vocab; }
size_t plan_of(int* ws, int n, int H, int vocab, Plan& p) {
  size_t at = 0;
  auto take = [&](size_t ints) { int* q = ws + at; at += round4(ints); return q; };
  p.cursor = take(4);
  p.count = take(vocab);
  p.begin = take(vocab);
  p.rank = take(n);
  p.pos = take(n);
  p.row = (int4*)take(4 * (size_t)rows_at_most(n, vocab));
  p.task = (int4*)take(4 * ((size_t)n * H / 16384 + n / (kFew + 1) + 1));
  p.most = take(n / (kMany + 1));
  p.parts = (float*)take((size_t)(n / (kMany + 1)) * kWindows * H);
  return at;
}

// The ordering's launches are short and leave most of the chip idle: each clears a part of the gradient on the side, in the workgroups behind its own.
struct Fill {
  float4* p;
  size_t from, to;  // in float4
  int own;          // the launch's workgroups before those that clear
};
__device__ __forceinline__ bool clears(const Fill& f) {
  if ((int)blockIdx.x < f.own) return false;
  const size_t step = (size_t)(gridDim.x - f.own) * blockDim.x;
  for (size_t i = f.from + (size_t)(blockIdx.x - f.own) * blockDim.x + threadIdx.x; i < f.to; i += step) f.p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  return true;
}

__global__ __launch_bounds__(256) void embed_clear_kernel(int4* p, size_t n4, const Fill fill) {
  if (clears(fill)) return;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (size_t)fill.own * 256) p[i] = make_int4(0, 0, 0, 0);
}

// Lanes of one id take their numbers with a single atomic (a batch of one repeated token would otherwise wait for n atomics on one address):
// every lane learns which lanes share its id, then the lowest of each such set asks for all of them, all sets at once.  (Looking at all 64 ids is
// worth it: with the first 8 looked at and the others asking for themselves, 32768 tokens of text took 15 us instead of 9.)
__global__ __launch_bounds__(256) void embed_rank_kernel(const Ids ids, int n, int vocab, int* __restrict__ count, int* __restrict__ rank,
                                                         const Fill fill) {
  if (clears(fill)) return;
  const int i = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 63;
  const long long id = i < n ? ids.at(i) : -1;
  const bool ok = id >= 0 && id < vocab;
  const int mine = ok ? (int)id : -1;
  uint64_t left = __ballot(ok), same = 1ull << lane;
  while (left) {
    const int v = __builtin_amdgcn_readlane(mine, (int)__builtin_ctzll(left));
    const uint64_t eq = __ballot(mine == v);
    if (mine == v) same = eq;
    left &= ~eq;
  }
  const int lead = (int)__builtin_ctzll(same);
  int base = 0;
  if (ok && lane == lead) base = atomicAdd(count + mine, (int)__popcll(same));
  base = __shfl(base, lead, 64);
  if (i < n) rank[i] = ok ? base + (int)__popcll(same & ((1ull << lane) - 1ull)) : -1;
}

// empty: rows without tokens are rows, too
__global__ __launch_bounds__(1024) void embed_alloc_kernel(const Plan p, int vocab, int H, int empty, const Fill fill) {
  __shared__ int part[2][17];
  if (clears(fill)) return;
  const int v = blockIdx.x * 1024 + threadIdx.x, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int c = v < vocab ? p.count[v] : -1;
  const bool row = c <= kFew && (c > 0 || (c == 0 && empty));
  int sum = max(c, 0);  // inclusive over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  const uint64_t rows = __ballot(row);
  if (lane == 63) {
    part[0][wid] = sum;
    part[1][wid] = (int)__popcll(rows);
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    int run = 0;
    for (int w = 0; w < 16; ++w) {
      const int x = part[threadIdx.x][w];
      part[threadIdx.x][w] = run;
      run += x;
    }
    part[threadIdx.x][16] = run ? atomicAdd(p.cursor + threadIdx.x, run) : 0;
  }
  __syncthreads();
  if (c < 0) return;
  const int at = part[0][16] + part[0][wid] + sum - c;
  p.begin[v] = at;
  if (row) p.row[part[1][16] + part[1][wid] + (int)__popcll(rows & ((1ull << lane) - 1ull))] = make_int4(v, c, at, 0);
  else if (c > kMany) p.most[atomicAdd(p.cursor + 3, 1)] = v;
  else if (c > kFew) {
    const int lanes = slice_lanes(c), log = 31 - __clz(lanes), slices = (H + lanes * 8 - 1) / (lanes * 8);
    const int first = atomicAdd(p.cursor + 2, slices);
    for (int k = 0; k < slices; ++k) p.task[first + k] = make_int4(v, c, at, k * lanes << 4 | log);
  }
}

__global__ __launch_bounds__(256) void embed_place_kernel(const Ids ids, int n, const int* __restrict__ begin, const int* __restrict__ rank, int* __restrict__ pos,
                                                          const Fill fill) {
  if (clears(fill)) return;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int r = rank[i];
  if (r >= 0) pos[begin[(int)ids.at(i)] + r] = i;
}

__device__ __forceinline__ void put4(float* out, size_t at, const float4& acc, float scale, int add) {
  float4 v = make_float4(acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale);
  if (add) {
    const float4 o = load4<true>(out, at);
    v = make_float4(fmaf(acc.x, scale, o.x), fmaf(acc.y, scale, o.y), fmaf(acc.z, scale, o.z), fmaf(acc.w, scale, o.w));
  }
  store4<true>(out, at, v);
}
__device__ __forceinline__ void put8(float* out, size_t at, const float (&acc)[8], float scale, int add) {
  put4(out, at, make_float4(acc[0], acc[1], acc[2], acc[3]), scale, add);
  put4(out, at + 4, make_float4(acc[4], acc[5], acc[6], acc[7]), scale, add);
}
__device__ __forceinline__ void add4(float4& a, const float4& x) { a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w; }

// one wave: columns col0 .. col0 + 511 of a table row of at most kFew tokens
template <bool F32>
__device__ void sum_few(const void* dout, float* out, int v, int c, const int* pos, int H, int col0, float scale, int add, int lane) {
  const int mine = lane < c ? pos[lane] : INT32_MAX;
  int smaller = 0;
  for (int j = 0; j < c; ++j) smaller += __builtin_amdgcn_readlane(mine, j) < mine;
  // lanes without a position go behind those with one, each to a lane of its own
  const int sorted = __builtin_amdgcn_ds_permute((lane < c ? smaller : lane) * 4, mine);
  // (the lanes behind the last column stay with the others, on column 0: a lane that is read from has to be active)
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
  if (col < H) put8(out, (size_t)v * H + col, acc, scale, add);
}

// one workgroup: the tokens of an id at positions [from, to), the 8 * lanes columns from col0.  The 256 / lanes groups of lanes take the ordered
// positions in turn; the groups' sums are joined in a fixed order, in the wave first and then over the waves.
template <bool F32>
__device__ void sum_many(const void* dout, float* dst, size_t dst_at, int c, const int* pos, int from, int to, int H, int col0, int lanes, float scale, int add,
                         uint32_t* map, int* list, float4* joined, int* counts) {
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int sub = tid & (lanes - 1), col = col0 + sub * 8, group = tid / lanes, groups = 256 / lanes;
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
        for (int j0 = group; j0 < got; j0 += 4 * groups) {
          float x[4][8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const bool is = j0 + u * groups < got;
            load8<F32>(dout, (size_t)list[is ? j0 + u * groups : j0] * H + col, x[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] = is ? x[u][e] : 0.f;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += x[u][e];
        }
    }
    __syncthreads();
  }
  for (int d = lanes; d < 64; d <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor(acc[e], d, 64);
  joined[tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  joined[256 + tid] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  __syncthreads();
  if (tid < lanes && col < H) {
    float4 a = joined[tid], b = joined[256 + tid];
    for (int t = tid + max(lanes, 64); t < 256; t += max(lanes, 64)) {
      add4(a, joined[t]);
      add4(b, joined[256 + t]);
    }
    put4(dst, dst_at + col, a, scale, add);
    put4(dst, dst_at + col + 4, b, scale, add);
  }
  __syncthreads();
}

template <bool F32>
__global__ __launch_bounds__(256, 6) void embed_sum_kernel(const void* __restrict__ dout, float* __restrict__ out, const Plan p, int n, int H, int vocab,
                                                        float scale, int add, int blocks_many) {
  __shared__ uint32_t map[kMap / 32];
  __shared__ int list[kBatch];
  __shared__ int counts[4];
  __shared__ float4 joined[512];
  if ((int)blockIdx.x < blocks_many) {  // the frequent ids first: their workgroups take longest
    const int slices = (H + kLeast * 8 - 1) / (kLeast * 8), window = (n + kWindows - 1) / kWindows;
    const long long split = (long long)p.cursor[3] * kWindows * slices, tasks = split + p.cursor[2];
    for (long long t = blockIdx.x; t < tasks; t += blocks_many) {
      if (t < split) {
        const int part = (int)(t / slices), v = p.most[part / kWindows], from = part % kWindows * window;
        sum_many<F32>(dout, p.parts, (size_t)part * H, p.count[v], p.pos + p.begin[v], from, min(from + window, n), H, (int)(t % slices) * kLeast * 8, kLeast, 1.0f, 0,
                      map, list, joined, counts);
      } else {
        const int4 k = p.task[t - split];
        sum_many<F32>(dout, out, (size_t)k.x * H, k.y, p.pos + k.z, 0, n, H, (k.w >> 4) * 8, 1 << (k.w & 15), scale, add, map, list, joined, counts);
      }
    }
    return;
  }
  const int parts = (H + kWide - 1) / kWide, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long items = (long long)p.cursor[1] * parts;
  for (long long i = (long long)((int)blockIdx.x - blocks_many) * 4 + wid; i < items; i += (long long)((int)gridDim.x - blocks_many) * 4) {
    const int4 k = p.row[i / parts];
    sum_few<F32>(dout, out, k.x, k.y, p.pos + k.z, H, (int)(i % parts) * kWide, scale, add, threadIdx.x & 63);
  }
}

__global__ __launch_bounds__(256) void embed_join_kernel(float* __restrict__ out, const Plan p, int H, float scale, int add) {
  for (int k = blockIdx.x; k < p.cursor[3]; k += gridDim.x)
    for (int col = threadIdx.x * 4; col < H; col += 1024) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < kWindows; ++w) add4(acc, load4<true>(p.parts, ((size_t)k * kWindows + w) * H + col));
      put4(out, (size_t)p.most[k] * H + col, acc, scale, add);
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
  // (2048 lanes' work a workgroup; more where a launch, which counts its work-items in 32 bits, could not have that many)
  const int per = std::max(std::max(1, 2048 / (H / 4)), (n + kGroups - 1) / kGroups);
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
  // (the launches clear in proportion to their own times, in elevenths)
  const bool early = !accumulate && clears_early(n, vocab);
  const size_t out4 = early ? (size_t)vocab * H / 4 : 0;
  const int fillers = early ? (int)std::min<size_t>(kFillers, out4 / 11 / 1024 + 1) : 0;  // workgroups of a launch that clear
  auto part = [&](int from, int to, int own) { return Fill{(float4*)dtable, out4 / 11 * from, to == 11 ? out4 : out4 / 11 * to, own}; };
  const size_t clear4 = (round4(4) + round4(vocab)) / 4;
  const int b_clear = (int)std::min<size_t>((clear4 + 255) / 256, 1024), b_ids = (n + 255) / 256, b_alloc = (vocab + 1023) / 1024;
  hipLaunchKernelGGL(embed_clear_kernel, dim3(b_clear + fillers), dim3(256), 0, st, (int4*)p.cursor, clear4, part(0, n == 0 ? 11 : 2, b_clear));
  if (n == 0) {
    CK_LAUNCH("embed_bwd(clear)");
    return COCODR_OK;
  }
  hipLaunchKernelGGL(embed_rank_kernel, dim3(b_ids + fillers), dim3(256), 0, st, d, n, vocab, p.count, p.rank, part(2, 6, b_ids));
  hipLaunchKernelGGL(embed_alloc_kernel, dim3(b_alloc + fillers / 4), dim3(1024), 0, st, p, vocab, H, !accumulate && !early, part(6, fillers >= 4 ? 9 : 6, b_alloc));
  hipLaunchKernelGGL(embed_place_kernel, dim3(b_ids + fillers), dim3(256), 0, st, d, n, p.begin, p.rank, p.pos, part(fillers >= 4 ? 9 : 6, 11, b_ids));
  CK_LAUNCH("embed_bwd(order)");
  const int blocks_many = (int)std::min<long long>(kTaskers, n > kFew ? (long long)n * H / 16384 + n / (kFew + 1) + 1 : 0);
  const long long waves = (long long)rows_at_most(n, vocab) * ((H + kWide - 1) / kWide);
  const dim3 grid((unsigned)(blocks_many + std::min<long long>(kRowers, (waves + 3) / 4)));
  if (dout_f32) hipLaunchKernelGGL(embed_sum_kernel<true>, grid, dim3(256), 0, st, dout, dtable, p, n, H, vocab, scale, accumulate, blocks_many);
  else hipLaunchKernelGGL(embed_sum_kernel<false>, grid, dim3(256), 0, st, dout, dtable, p, n, H, vocab, scale, accumulate, blocks_many);
  if (n > kMany) hipLaunchKernelGGL(embed_join_kernel, dim3(std::min(1024, n / (kMany + 1))), dim3(256), 0, st, dtable, p, H, scale, accumulate);
  CK_LAUNCH("embed_bwd");
  return COCODR_OK;
}
