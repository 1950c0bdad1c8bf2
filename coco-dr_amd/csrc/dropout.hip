// Dropout as an operator of its own, with the generator and the mask of the fused sites (include/cocodr.h "Dropout"): the mask is a hash
// of the element's flat index, so it is computed where it is needed, forward and backward, and never stored.
//   out_i = keep(i) ? scale x_i : 0   (+ r_i),  in fp32, rounded once.
// Bound by memory: x (and r) in, out out.  A hash serves two elements and costs two 32-bit multiplications (quarter rate) and six other
// integer operations - about a fifth of the time that the elements' 4 to 8 bytes each take.
#include "common.h"

namespace {

// elements a thread takes at once: 16 bytes, so that a wave's access is whole lines
template <bool F32> constexpr int kPer = F32 ? 4 : 8;

template <bool F32> struct Elem;
template <> struct Elem<false> {
  typedef uint16_t T;
  static __device__ __forceinline__ void load(const T* p, float (&v)[8]) { unpack8(*reinterpret_cast<const uint4*>(p), v); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[8]) { *reinterpret_cast<uint4*>(p) = pack8(v); }
  static __device__ __forceinline__ float load(const T* p) { return bf2f(*p); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = f2bf(v); }
};
template <> struct Elem<true> {
  typedef float T;
  static __device__ __forceinline__ void load(const T* p, float (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
};

// WIDE: all pointers are 16-byte aligned (a contiguous view into a larger tensor may begin anywhere: 16384 x 4096 from an odd element on 111 us in
// bf16 and 142 in fp32, aligned 38 and 94); what is left of n goes one by one
template <bool F32, bool ADD, bool WIDE>
__global__ __launch_bounds__(256) void dropout_kernel(const void* x_, const void* r_, void* out_, size_t n, const cocodr_dropout_mask dm) {
  typedef Elem<F32> E;
  const typename E::T *x = (const typename E::T*)x_, *r = (const typename E::T*)r_;
  typename E::T* out = (typename E::T*)out_;
  constexpr int PER = kPer<F32>;
  for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * PER; i < n; i += (size_t)gridDim.x * 256 * PER) {
    float v[PER], w[PER];
    const bool whole = i + PER <= n;
    if (WIDE && whole) {
      E::load(x + i, v);
      if constexpr (ADD) E::load(r + i, w);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        v[e] = i + e < n ? E::load(x + i + e) : 0.f;
        if constexpr (ADD) w[e] = i + e < n ? E::load(r + i + e) : 0.f;
      }
    }
    drop_apply<PER>(v, i, dm);
    if constexpr (ADD) {
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] += w[e];
    }
    if (WIDE && whole) E::store(out + i, v);
    else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (i + e < n) E::store(out + i + e, v[e]);
    }
  }
}

template <bool F32, bool ADD>
void launch(const void* x, const void* r, void* out, size_t n, const cocodr_dropout_mask& dm, hipStream_t st) {
  const bool wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(r) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const size_t groups = (n + 256 * kPer<F32> - 1) / (256 * kPer<F32>);
  const dim3 grid((unsigned)(groups < 65536 ? groups : 65536));
  if (wide) hipLaunchKernelGGL((dropout_kernel<F32, ADD, true>), grid, dim3(256), 0, st, x, r, out, n, dm);
  else hipLaunchKernelGGL((dropout_kernel<F32, ADD, false>), grid, dim3(256), 0, st, x, r, out, n, dm);
}

int run(const char* what, const void* x, const void* r, void* out, size_t n, int f32, const cocodr_dropout_mask* drop, hipStream_t st) {
  CK_ARG(drop, "%s: null mask", what);
  CK_ARG(drop->threshold < 65536, "%s: threshold %u: below 65536 is wanted", what, drop->threshold);
  CK_ARG(n <= (1ull << 33), "%s: %zu elements: the mask's generator counts 2^32 pairs", what, n);
  if (n == 0) return COCODR_OK;
  CK_ARG(x && out, "%s: null pointer", what);
  const uintptr_t part = f32 ? 3 : 1;
  CK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(r) | reinterpret_cast<uintptr_t>(out)) & part) == 0, "%s: pointers must be aligned to an element", what);
  if (f32) r ? launch<true, true>(x, r, out, n, *drop, st) : launch<true, false>(x, r, out, n, *drop, st);
  else r ? launch<false, true>(x, r, out, n, *drop, st) : launch<false, false>(x, r, out, n, *drop, st);
  CK_LAUNCH(what);
  return COCODR_OK;
}

}  // namespace

extern "C" int cocodr_dropout_fwd(const void* x, const void* residual, void* out, size_t n, int f32, const cocodr_dropout_mask* drop, cocodr_stream_t stream) {
  return run("dropout_fwd", x, residual, out, n, f32, drop, (hipStream_t)stream);
}
extern "C" int cocodr_dropout_bwd(const void* dout, void* dx, size_t n, int f32, const cocodr_dropout_mask* drop, cocodr_stream_t stream) {
  return run("dropout_bwd", dout, nullptr, dx, n, f32, drop, (hipStream_t)stream);
}
