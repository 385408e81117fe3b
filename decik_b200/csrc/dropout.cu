// Dropout from a counter-based generator (philox.cuh), with no stored mask: out = [residual +]
// keep * scale * x over n values in row-major order. The same call on the gradient is its backward.
//
// HBM-bound: each value is read once and written once, the mask is computed. 16,384 x 1536 bf16 added to an
// fp32 residual: 252 MB in 41.1 us (6.1 TB/s, 0.93 of a plain copy's rate); 830 x 1536 fp16: 2.8 us.
#include "philox.cuh"

namespace decik {
namespace {

template <typename X> __device__ __forceinline__ float load1(const X* p) { return Dt<X>::to_f(*p); }
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <typename X> __device__ __forceinline__ void store1(X* p, float v) { *p = Dt<X>::from_f(v); }
template <> __device__ __forceinline__ void store1<float>(float* p, float v) { *p = v; }

// 8 consecutive values as they lie in memory, one or two 16-byte pieces
template <typename X>
struct Eight {
  uint4 v[sizeof(X) / 2];
  __device__ __forceinline__ void load(const X* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(X) / 2); ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    if constexpr (sizeof(X) == 2) {
      unpack8<X>(v[0], f);
    } else {
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    }
  }
};
template <typename O>
__device__ __forceinline__ void store8(O* p, const float (&f)[8]) {
  if constexpr (sizeof(O) == 2) {
    stg16(p, pack8<O>(f));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// A thread takes groups of 8 values, kUnroll of them with their loads in flight together (the residual
// case above: 43.4 us with 1, 41.1 with 2, 41.6 with 4). VEC: every pointer is 16-byte aligned; without
// it (122 us instead of 43 in a stream), and for the last n % 8 values, one value at a time. Dropped values
// are 0 whatever x holds there (NaN included).
constexpr int kUnroll = 2;

template <typename X, typename O, bool RES, bool VEC>
__global__ void __launch_bounds__(256)
dropout_kernel(const X* x, const O* residual, O* out, int64_t n, uint32_t cut, float scale,
               const int64_t* __restrict__ rng, int64_t stream_id) {
  const philox::Key key = philox::make_key(rng);
  const philox::Stream ctr = philox::make_stream(rng, stream_id);
  const int64_t groups = (n + 7) / 8, whole = VEC ? n / 8 : 0;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  int64_t g = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if constexpr (VEC) {
    for (; g < whole; g += kUnroll * stride) {
      Eight<X> xv[kUnroll];
      Eight<O> rv[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (g + u * stride < whole) {
          xv[u].load(x + 8 * (g + u * stride));
          if constexpr (RES) rv[u].load(residual + 8 * (g + u * stride));
        }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = g + u * stride;
        if (i >= whole) break;
        const uint4 w = philox::words(key, ctr, static_cast<unsigned long long>(i));
        float f[8], o[8] = {};
        xv[u].values(f);
        if constexpr (RES) rv[u].values(o);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = philox::keep_lane(w, j, cut) ? f[j] * scale : 0.f;
          o[j] = RES ? o[j] + v : v;
        }
        store8(out + 8 * i, o);
      }
    }
    g = whole + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;  // the last group, if it is not whole
  }
  for (; g < groups; g += stride) {
    const uint4 w = philox::words(key, ctr, static_cast<unsigned long long>(g));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = 8 * g + j;
      if (i >= n) break;
      float v = philox::keep_lane(w, j, cut) ? load1(x + i) * scale : 0.f;
      if constexpr (RES) v += load1(residual + i);
      store1(out + i, v);
    }
  }
}

template <typename X, typename O>
int launch(const void* x, const void* residual, void* out, int64_t n, double p, const int64_t* rng, int64_t stream_id,
           cudaStream_t s) {
  const uint32_t cut = philox::cut_of(p);
  const float scale = philox::scale_of(cut);
  const int64_t want = ((n + 7) / 8 + 255) / 256, cap = static_cast<int64_t>(sm_count()) * 16;
  const int grid = static_cast<int>(want < cap ? want : cap);
  const bool vec = aligned16(x) && aligned16(out) && (residual == nullptr || aligned16(residual));
  auto go = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(static_cast<const X*>(x), static_cast<const O*>(residual), static_cast<O*>(out), n, cut,
                                scale, rng, stream_id);
  };
  if (residual != nullptr) vec ? go(dropout_kernel<X, O, true, true>) : go(dropout_kernel<X, O, true, false>);
  else vec ? go(dropout_kernel<X, O, false, true>) : go(dropout_kernel<X, O, false, false>);
  return check_launch("dropout");
}

template <typename X>
int launch_x(int out_dtype, const void* x, const void* residual, void* out, int64_t n, double p, const int64_t* rng,
             int64_t stream_id, cudaStream_t s) {
  if (out_dtype == DECIK_F32) return launch<X, float>(x, residual, out, n, p, rng, stream_id, s);
  if (out_dtype == DECIK_BF16) return launch<X, __nv_bfloat16>(x, residual, out, n, p, rng, stream_id, s);
  return launch<X, __half>(x, residual, out, n, p, rng, stream_id, s);
}

bool valid_dtype(int d) { return d == DECIK_F16 || d == DECIK_BF16 || d == DECIK_F32; }

}  // namespace
}  // namespace decik

extern "C" int decik_dropout(const void* x, int x_dtype, const void* residual, void* out, int out_dtype, int64_t n,
                             double p, const int64_t* rng, int64_t stream_id, void* stream) {
  using namespace decik;
  if (n < 0) return set_error(DECIK_ERR_INVALID, "dropout: n=%lld", (long long)n);
  if (!philox::valid_p(p)) return set_error(DECIK_ERR_INVALID, "dropout: p=%g is not in [0, 1]", p);
  if (!valid_dtype(x_dtype) || !valid_dtype(out_dtype))
    return set_error(DECIK_ERR_INVALID, "dropout: dtypes %d -> %d are not F16/BF16/F32", x_dtype, out_dtype);
  if (n == 0) return DECIK_OK;
  if (!x || !out || !rng) return set_error(DECIK_ERR_INVALID, "dropout: null pointer");
  if (!aligned_to(x, dtype_bytes(x_dtype)) || !aligned_to(out, dtype_bytes(out_dtype)) ||
      !aligned_to(residual, dtype_bytes(out_dtype)) || !aligned_to(rng, 8))
    return set_error(DECIK_ERR_INVALID, "dropout: a pointer is not aligned to its values");
  cudaStream_t s = as_stream(stream);
  if (x_dtype == DECIK_F32) return launch_x<float>(out_dtype, x, residual, out, n, p, rng, stream_id, s);
  if (x_dtype == DECIK_BF16) return launch_x<__nv_bfloat16>(out_dtype, x, residual, out, n, p, rng, stream_id, s);
  return launch_x<__half>(out_dtype, x, residual, out, n, p, rng, stream_id, s);
}
