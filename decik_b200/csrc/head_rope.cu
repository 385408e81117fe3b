// The norm of each query and key head with the position rotation in the same pass, and the rotation
// by positions of several axes (time, height, width), forward and backward. For one head's row
// x = q (+ q_lora) of one token (D = head_dim, R = rotary_dim, j < R / 2):
//   r = rsqrt(mean(x^2) + eps),  y = x r w                      (without norms: y = x)
//   out[j] = y[j] cos[j] - y[j + R/2] sin[j],  out[j + R/2] = y[j + R/2] cos[j + R/2] + y[j] sin[j + R/2],
//   out[d] = y[d] for d >= R;
// backward, with g the transposed rotation of the gradient:
//   dw = sum over tokens and heads of g x r,  z = g w,  dx = r (z - x r^2 mean(z x)).
// The cosines come from fp32 tables [T, R] or, for several axes, from the token's positions:
// angle j = position[axis of j] * inv_freq[j].
//
// All arithmetic is fp32 with one rounding at the end. HBM-bound. L lanes hold a token's row of D values,
// 16 each, and walk over its heads: the angles (read from the tables or computed), with the weights
// folded in, stay in registers for all of them, a row's mean square is log2 L shuffles, and a lane's two
// 16-byte pieces are rotation partners. Norms and tables at 131,072 tokens, 28 / 4 heads of 128: 343 us for
// 2.28 GB, a plain copy's rate; three axes at 16,384 tokens, 12 / 2 heads: 20.0 us for 118 MB (5.9 TB/s);
// norm backward there: 36.9 us for 193 MB (5.2 TB/s; the pass itself 6 TB/s, then the weights' gradients).
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace decik {
namespace headrope {
namespace {

// where the angles come from: tables, or positions of up to four axes with the axis of each
// frequency in two bits
struct Angles {
  const float* cos;
  const float* sin;
  const void* pos;
  int pos32, n_axes;
  int64_t ld_pos;
  const float* inv_freq;
  uint32_t axis[8];
};

struct Args {
  decik_tensor3 q, ql, k;          // forward inputs; in the backward the saved ones
  decik_tensor3 gq, gk;            // backward: gradients
  decik_tensor3_mut oq, ok;        // forward: outputs; backward: dq, dk
  const void* wq;
  const void* wk;
  float* part;                     // backward: [CTA][2][D] partial sums of the weight gradients
  Angles ang;
  int64_t n_tok;
  int hq, hk, D, R;
  float eps;
};

__device__ __forceinline__ float load_w(const void* w, int dtype, int i) {
  return dtype == DECIK_F32 ? __ldg(static_cast<const float*>(w) + i)
         : dtype == DECIK_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i])
                               : __half2float(static_cast<const __half*>(w)[i]);
}

// cos and sin of position * inv_freq, to fp32's last bits of the exact product's: the quarter turns
// are counted and taken off in 64 bits (a far position times a 24-bit frequency needs more than 32),
// so that what is rounded to fp32 is at most an eighth of a turn, exact relative to itself. Adding
// 1.5 2^52 rounds to whole quarters and leaves their count in the sum's low bits (up to 2^51 quarters,
// beyond which 64 bits hold no angle).
__device__ __forceinline__ void sincos_of(double pos, float inv_freq, float& s, float& c) {
  const double quarters = pos * static_cast<double>(inv_freq) * 0.63661977236758134;  // 2 / pi
  const double whole = quarters + 6755399441055744.0;
  const int quadrant = __double2loint(whole);
  float a, b;
  sincospif(0.5f * static_cast<float>(quarters - (whole - 6755399441055744.0)), &a, &b);
  s = quadrant & 1 ? b : a;
  c = quadrant & 1 ? a : b;
  if (quadrant & 2) s = -s;
  if ((quadrant + 1) & 2) c = -c;
}

__device__ __forceinline__ double position(const Angles& a, int axis, int64_t t) {
  const int64_t i = axis * a.ld_pos + t;
  return a.pos32 ? static_cast<double>(__ldg(static_cast<const int*>(a.pos) + i))
                 : static_cast<double>(__ldg(static_cast<const long long*>(a.pos) + i));
}

// A row of D values is held by L lanes (4, 8 or 16: a power of two at or above D / 16), 16 values each:
// lane c holds the 8 values from lo and the 8 from hi. Lanes below R / 16 hold rotation partners (hi = lo
// + R / 2), those below D / 16 the values behind R, the rest nothing.
struct Lane {
  int lo, hi;
  bool active, rot;
};
__device__ __forceinline__ Lane lane_of(int c, int D, int R) {
  Lane l;
  l.rot = 16 * c < R;
  l.active = 16 * c < D;
  l.lo = l.rot ? 8 * c : 16 * c;
  l.hi = l.rot ? R / 2 + 8 * c : 16 * c + 8;
  return l;
}

__device__ __forceinline__ void load8f(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// cos and sin of the lane's values at token t: of its lo and hi values from tables, of its frequencies
// (the same for both) from positions; 1 and 0 for values that are not rotated. N = 8 or 16.
template <bool AXES>
__device__ __forceinline__ void load_angles(const Args& p, const Lane& l, bool ok, int64_t t,
                                            float (&c)[AXES ? 8 : 16], float (&s)[AXES ? 8 : 16]) {
#pragma unroll
  for (int i = 0; i < (AXES ? 8 : 16); ++i) c[i] = 1.f, s[i] = 0.f;
  if (!ok || !l.rot) return;
  if constexpr (AXES) {
    double pos[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) pos[a] = a < p.ang.n_axes ? position(p.ang, a, t) : 0.0;
    float f[8];
    load8f(p.ang.inv_freq + l.lo, f);
    const uint32_t map = p.ang.axis[l.lo >> 4] >> (2 * (l.lo & 15));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int axis = (map >> (2 * i)) & 3;
      const double x = axis & 2 ? (axis & 1 ? pos[3] : pos[2]) : (axis & 1 ? pos[1] : pos[0]);
      sincos_of(x, f[i], s[i], c[i]);
    }
  } else {
    float v[4][8];
    load8f(p.ang.cos + t * p.R + l.lo, v[0]);
    load8f(p.ang.cos + t * p.R + l.hi, v[1]);
    load8f(p.ang.sin + t * p.R + l.lo, v[2]);
    load8f(p.ang.sin + t * p.R + l.hi, v[3]);
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = v[0][i], c[8 + i] = v[1][i], s[i] = v[2][i], s[8 + i] = v[3][i];
  }
}

// the lane's 16 weights (lo, then hi); zeros in lanes that hold nothing
__device__ __forceinline__ void load_weights(const void* w, int dtype, const Lane& l, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = l.active ? load_w(w, dtype, l.lo + i) : 0.f;
    v[8 + i] = l.active ? load_w(w, dtype, l.hi + i) : 0.f;
  }
}

template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Raw {  // a lane's 16 values of a row as they lie in memory
  uint4 lo, hi;
};
template <typename T>
__device__ __forceinline__ Raw load_raw(const T* p, const Lane& l, bool ok) {
  Raw r{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  if (ok) {
    r.lo = ldg16(p + l.lo);
    r.hi = ldg16(p + l.hi);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack(const Raw& r, float (&x)[16]) {
  float a[8], b[8];
  unpack8<T>(r.lo, a);
  unpack8<T>(r.hi, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = a[i], x[8 + i] = b[i];
}
template <typename T>
__device__ __forceinline__ void add(const Raw& r, float (&x)[16]) {
  float y[16];
  unpack<T>(r, y);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] += y[i];
}
template <typename T>
__device__ __forceinline__ void store(T* p, const Lane& l, const float (&x)[16]) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = x[i], b[i] = x[8 + i];
  stg16(p + l.lo, pack8<T>(a));
  stg16(p + l.hi, pack8<T>(b));
}

constexpr int kThreads = 128;

// Forward; with sign -1 and without norms also the backward (the rotation by the opposite angle).
// Block (x, y): 128 / L tokens, heads y * per_group .. of the queries' and then the keys' heads. The
// loads of U heads are in flight together: 343 us at 131,072 tokens with 4, 494 with 2, 361 with 8; with
// a LoRA delta, which doubles the loads, 10.4 us at 4,099 tokens with 2, 11.7 with 1, 15.7 with 4.
// PART: R < D. A value behind R is no partner of another, and a sine of 0 would not keep an infinity or a NaN
// there from it (0 inf is NaN), so its partner's share is left out: by a select of each value without norms
// (6.8 us instead of 6.5 at 4,099 tokens of 14 / 2 heads of 80, none of it at 16,384 of 12 / 2 of 128). With norms
// the selects took 28.6 us instead of 24.3 at 16,384 of 12 / 2 of 128 (R = 64), a branch on the lane as much; there
// only a row with an infinity comes to that (its r is 0, and 0 inf is NaN), which is read again: 24.7 us.
template <typename T, int L, bool NORM, bool AXES, bool LORA, bool PART>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args p, int w_dtype, int per_group, float sign) {
  constexpr int U = LORA ? 2 : 4;
  const Lane l = lane_of(threadIdx.x % L, p.D, p.R);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  const bool ok = t < p.n_tok && l.active;
  const int h0 = blockIdx.y * per_group, h1 = h0 + per_group < p.hq + p.hk ? h0 + per_group : p.hq + p.hk;
  const float inv_d = 1.f / static_cast<float>(p.D);
  float cs[AXES ? 8 : 16], sn[AXES ? 8 : 16];
  load_angles<AXES>(p, l, ok, t, cs, sn);
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {  // queries, keys
    const int first = part ? (h0 > p.hq ? h0 - p.hq : 0) : h0, last = part ? h1 - p.hq : (h1 < p.hq ? h1 : p.hq);
    if (first >= last) continue;
    const decik_tensor3& in = part ? p.k : p.q;
    const decik_tensor3_mut& out = part ? p.ok : p.oq;
    // out[lo] = r (x[lo] m[0] - x[hi] m[1]), out[hi] = r (x[hi] m[2] + x[lo] m[3])
    float m[4][8], w[16];
    if constexpr (NORM) load_weights(part ? p.wk : p.wq, w_dtype, l, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int hi = AXES ? i : 8 + i;
      m[0][i] = NORM ? w[i] * cs[i] : cs[i];
      m[1][i] = PART && !l.rot ? 0.f : sign * (NORM ? w[8 + i] * sn[i] : sn[i]);
      m[2][i] = NORM ? w[8 + i] * cs[hi] : cs[hi];
      m[3][i] = PART && !l.rot ? 0.f : sign * (NORM ? w[i] * sn[hi] : sn[hi]);
    }
    const T* src = static_cast<const T*>(in.ptr) + t * in.tok_stride + first * in.head_stride;
    const T* lora = LORA && !part ? static_cast<const T*>(p.ql.ptr) + t * p.ql.tok_stride + first * p.ql.head_stride : src;
    const int64_t lora_hs = LORA && !part ? p.ql.head_stride : 0;
    T* dst = static_cast<T*>(out.ptr) + t * out.tok_stride + first * out.head_stride;
    for (int h = first; h < last; h += U) {
      Raw raw[U], rl[LORA ? U : 1];
      unsigned infinite = 0u;  // a bit for each row whose r is 0, in lanes behind R
#pragma unroll
      for (int u = 0; u < U; ++u) {
        raw[u] = load_raw(src + u * in.head_stride, l, ok && h + u < last);
        if constexpr (LORA) rl[u] = load_raw(lora + u * lora_hs, l, ok && !part && h + u < last);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u >= last) break;
        float x[16], o[16], r = 1.f;
        unpack<T>(raw[u], x);
        if constexpr (LORA) add<T>(rl[u], x);
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
          r = rsqrtf(row_sum<L>(ss) * inv_d + p.eps);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= r;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i] = x[i] * m[0][i] - (PART && !NORM && !l.rot ? 0.f : x[8 + i]) * m[1][i];
          o[8 + i] = x[8 + i] * m[2][i] + (PART && !NORM && !l.rot ? 0.f : x[i]) * m[3][i];
        }
        const bool later = NORM && PART && !l.rot && r == 0.f;
        if constexpr (NORM && PART) infinite |= (later ? 1u : 0u) << u;
        if (ok && !later) store(dst + u * out.head_stride, l, o);
      }
      if constexpr (NORM && PART) {
        if (infinite != 0u && ok) {  // values behind R of rows with an infinity, each alone
#pragma unroll 1
          for (int u = 0; u < U; ++u) {
            if (!(infinite >> u & 1u)) continue;
            float x[16];
            unpack<T>(load_raw(src + u * in.head_stride, l, true), x);
            if constexpr (LORA) add<T>(load_raw(lora + u * lora_hs, l, !part), x);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = x[i] * 0.f * (i < 8 ? m[0][i & 7] : m[2][i & 7]);
            store(dst + u * out.head_stride, l, x);
          }
        }
      }
      src += U * in.head_stride;
      lora += U * lora_hs;
      dst += U * out.head_stride;
    }
  }
}

// Pairs of fp32 values in one register pair and instruction (the packed arithmetic of sm_100; each half
// rounds as the single instruction does).
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2f(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2f(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float sum2(f2 v) {
  float x, y;
  unpack2f(v, x, y);
  return x + y;
}
// 8 16-bit values as 4 pairs, and back
template <typename T>
__device__ __forceinline__ void unpack_f2(const uint4& v, f2* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2f(Dt<T>::lo_f(w[i]), Dt<T>::hi_f(w[i]));
}
template <typename T>
__device__ __forceinline__ uint4 pack_f2(const f2* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpack2f(x[i], a, b);
    w[i] = Dt<T>::pack2(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The backward with norms. The rows (tile of 32 / L tokens, head) in tile order are shared out evenly over
// the warps, each a contiguous range: a warp's lanes keep a tile's angles while its heads last. A row's
// bytes (gradient, input) are on their way kDepth - 1 rows ahead through cp.async into slots of the
// lane's own, across heads and tiles. The weight gradients are summed in fp32: a lane's own rows in
// registers (kept in a slot in shared memory while the warp is at the other part, queries or keys),
// then the CTA's lanes that hold the same values, then the CTAs in a kernel of their own, all in a
// fixed order.
// Two rows ahead take 37.1 us at 16,384 tokens of 12 / 2 heads, three 37.6; a tile a CTA at a time, with a
// row ahead in registers, took 48.2. PART as in the forward, by selects (10,007 tokens of 16 / 4 heads of 64, R =
// 32: 22.0 us instead of 21.6).
constexpr int kDepth = 3, kSlot = 20;  // kSlot: floats of a lane's slot, 16 and padding against bank conflicts

template <int L, bool LORA>
constexpr int bwd_smem() {
  return kThreads * kDepth * (LORA ? 6 : 4) * 16 + (2 * kThreads + 2 * L) * kSlot * 4;
}

template <typename T, int L, bool AXES, bool LORA, bool PART>
__global__ void __launch_bounds__(kThreads, LORA ? 3 : 4) norm_bwd_kernel(const Args p, int w_dtype, int64_t n_rows, int64_t per_warp) {
  constexpr int P = LORA ? 6 : 4, TOK = 32 / L;
  extern __shared__ __align__(16) unsigned char smem[];
  float* const slots = reinterpret_cast<float*>(smem + kThreads * kDepth * P * 16);  // [2][kThreads][kSlot]
  float* const ws = slots + 2 * kThreads * kSlot;                                    // [2][L][kSlot]: weights
  const int lane = threadIdx.x & 31, c = threadIdx.x % L, heads = p.hq + p.hk;
  const Lane l = lane_of(c, p.D, p.R);
  if (threadIdx.x < 2 * L) {
    float w[16];
    load_weights(threadIdx.x < L ? p.wq : p.wk, w_dtype, l, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) ws[threadIdx.x * kSlot + i] = w[i];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) slots[(j * kThreads + threadIdx.x) * kSlot + i] = 0.f;
  __syncthreads();
  // the warp's number broadcast, so that the row's state below lives in uniform registers
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int64_t row0 = warp * per_warp;
  int left = static_cast<int>(n_rows - row0 < per_warp ? n_rows - row0 : per_warp);
  const float inv_d = 1.f / static_cast<float>(p.D);
  f2 dw[8] = {};
  int part = 0;
  if (left > 0) {
    // The row read next: its tile, head and running addresses, set anew where a part begins. A lane
    // without a value of its own (beyond the tokens, or D) reads nothing, from an address that is there.
    const int tile0 = static_cast<int>(row0 / heads), n_tok = static_cast<int>(p.n_tok);
    const int off = l.active ? l.lo : 0, up = l.active ? l.hi - l.lo : 0;
    int h = static_cast<int>(row0 - static_cast<int64_t>(tile0) * heads);
    int fh = h, to_read = left, ft = tile0 * TOK + lane / L;
    const T *g, *x, *y = nullptr;
    const uint32_t ring_at = ptx::smem_u32(smem + threadIdx.x * 16);  // piece q of stage s at (s P + q) kThreads 16
    auto seek = [&]() {
      const int64_t t = ft < n_tok ? ft : n_tok - 1;
      const bool k = fh >= p.hq;
      const int hh = k ? fh - p.hq : fh;
      const decik_tensor3& gr = k ? p.gk : p.gq;
      const decik_tensor3& in = k ? p.k : p.q;
      g = static_cast<const T*>(gr.ptr) + t * gr.tok_stride + hh * gr.head_stride + off;
      x = static_cast<const T*>(in.ptr) + t * in.tok_stride + hh * in.head_stride + off;
      if constexpr (LORA) y = static_cast<const T*>(p.ql.ptr) + t * p.ql.tok_stride + (k ? 0 : hh * p.ql.head_stride) + off;
    };
    seek();
    auto fetch = [&](int stage) {
      if (to_read > 0) {
        const uint32_t dst = ring_at + stage * (P * kThreads * 16);
        const bool there = ft < n_tok && l.active, k = fh >= p.hq;
        ptx::cp_async16(dst, g, there);
        ptx::cp_async16(dst + kThreads * 16, g + up, there);
        ptx::cp_async16(dst + 2 * kThreads * 16, x, there);
        ptx::cp_async16(dst + 3 * kThreads * 16, x + up, there);
        if constexpr (LORA) {
          ptx::cp_async16(dst + 4 * kThreads * 16, y, there && !k);
          ptx::cp_async16(dst + 5 * kThreads * 16, y + up, there && !k);
          if (!k && fh + 1 < p.hq) y += p.ql.head_stride;
        }
        ++fh;
        --to_read;
        if (fh == heads) fh = 0, ft += TOK;
        if (fh == 0 || fh == p.hq) {
          seek();
        } else {
          g += k ? p.gk.head_stride : p.gq.head_stride;
          x += k ? p.k.head_stride : p.q.head_stride;
        }
      }
      ptx::cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kDepth - 1; ++s) fetch(s);
    int t = tile0 * TOK + lane / L;
    bool ok = t < n_tok && l.active;
    // cos of the lane's lo and hi pairs, sin of hi, - sin of lo
    f2 cl[4], ch[AXES ? 1 : 4], sh[4], nsl[4];
    auto angles = [&]() {
      float cs[AXES ? 8 : 16], sn[AXES ? 8 : 16];
      load_angles<AXES>(p, l, ok, t, cs, sn);
      constexpr int H = AXES ? 0 : 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cl[i] = pack2f(cs[2 * i], cs[2 * i + 1]);
        if constexpr (!AXES) ch[i] = pack2f(cs[H + 2 * i], cs[H + 2 * i + 1]);
        sh[i] = pack2f(sn[H + 2 * i], sn[H + 2 * i + 1]);
        nsl[i] = pack2f(-sn[2 * i], -sn[2 * i + 1]);
      }
    };
    auto swap = [&](int to) {  // the sums of one part to their slot, those of the other from theirs
      f2* const a = reinterpret_cast<f2*>(slots + (part * kThreads + threadIdx.x) * kSlot);
      const f2* const b = reinterpret_cast<const f2*>(slots + (to * kThreads + threadIdx.x) * kSlot);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = dw[i];
        dw[i] = b[i];
      }
      part = to;
    };
    T* dst;  // the result's running address
    auto aim = [&]() {
      const decik_tensor3_mut& out = h >= p.hq ? p.ok : p.oq;
      dst = static_cast<T*>(out.ptr) + t * out.tok_stride + (h >= p.hq ? h - p.hq : h) * out.head_stride + off;
    };
    angles();
    aim();
    for (int stage = 0; left > 0; --left) {
      ptx::cp_async_wait<kDepth - 2>();
      __syncwarp();  // keeps the reads below behind the wait
      fetch(stage == 0 ? kDepth - 1 : stage - 1);
      if ((h >= p.hq) != (part == 1)) swap(part ^ 1);
      const unsigned char* const got = smem + threadIdx.x * 16 + stage * (P * kThreads * 16);
      f2 v[8], z[8];
      {
        f2 gv[8];
        unpack_f2<T>(*reinterpret_cast<const uint4*>(got), gv);
        unpack_f2<T>(*reinterpret_cast<const uint4*>(got + kThreads * 16), gv + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[i] = fma2(gv[i], cl[i], mul2(!PART || l.rot ? gv[4 + i] : 0ull, sh[i]));
          z[4 + i] = fma2(gv[4 + i], AXES ? cl[i] : ch[AXES ? 0 : i], mul2(!PART || l.rot ? gv[i] : 0ull, nsl[i]));
        }
      }
      unpack_f2<T>(*reinterpret_cast<const uint4*>(got + 2 * kThreads * 16), v);
      unpack_f2<T>(*reinterpret_cast<const uint4*>(got + 3 * kThreads * 16), v + 4);
      if constexpr (LORA) {
        f2 yv[8];
        unpack_f2<T>(*reinterpret_cast<const uint4*>(got + 4 * kThreads * 16), yv);
        unpack_f2<T>(*reinterpret_cast<const uint4*>(got + 5 * kThreads * 16), yv + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = add2(v[i], yv[i]);
      }
      // Both sums in one round of shuffles: of x^2, and of z w x with x as it was read (the mean needs it
      // times r, which the first sum gives).
      f2 ss0 = mul2(v[0], v[0]), ss1 = mul2(v[1], v[1]), zx0 = 0ull, zx1 = 0ull;  // two zeros each
      f2 d[8];
      const ulonglong2* const w = reinterpret_cast<const ulonglong2*>(ws + (part * L + c) * kSlot);
#pragma unroll
      for (int i = 2; i < 8; i += 2) {
        ss0 = fma2(v[i], v[i], ss0);
        ss1 = fma2(v[i + 1], v[i + 1], ss1);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const ulonglong2 wv = w[i / 2];
        d[i] = mul2(z[i], v[i]);
        d[i + 1] = mul2(z[i + 1], v[i + 1]);
        zx0 = fma2(d[i], wv.x, zx0);
        zx1 = fma2(d[i + 1], wv.y, zx1);
        z[i] = mul2(z[i], wv.x);
        z[i + 1] = mul2(z[i + 1], wv.y);
      }
      float ss = sum2(add2(ss0, ss1)), zx = sum2(add2(zx0, zx1));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        zx += __shfl_xor_sync(0xffffffffu, zx, o);
      }
      // (of a row that is not there 0, so that it adds nothing to the sums with eps = 0 either)
      const float rs = rsqrtf(ss * inv_d + p.eps), r = t < n_tok ? rs : 0.f, mean = -(r * r) * (zx * inv_d);
      const f2 rr = pack2f(r, r), mm = pack2f(mean, mean);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[i] = fma2(d[i], rr, dw[i]);
        z[i] = mul2(rr, fma2(v[i], mm, z[i]));
      }
      if (ok) {
        stg16(dst, pack_f2<T>(z));
        stg16(dst + up, pack_f2<T>(z + 4));
      }
      if (++h == heads) {
        h = 0;
        t += TOK;
        ok = t < n_tok && l.active;
        if (left > 1) angles();
      }
      if (h == 0 || h == p.hq) aim();
      else dst += part ? p.ok.head_stride : p.oq.head_stride;
      stage = stage + 1 == kDepth ? 0 : stage + 1;
    }
    swap(part ^ 1);  // the last sums to their slot
  }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * 16 * L; j += kThreads) {  // value i of lane k over the CTA's rows
    const int q = j / (16 * L), k = j / 16 % L, i = j % 16;
    const Lane o = lane_of(k, p.D, p.R);
    float s = 0.f;
    for (int n = k; n < kThreads; n += L) s += slots[(q * kThreads + n) * kSlot + i];
    if (o.active) p.part[(2 * static_cast<int64_t>(blockIdx.x) + q) * p.D + (i < 8 ? o.lo + i : o.hi + i - 8)] = s;
  }
}

// dw[d] = the sum of the CTAs' partials in a fixed order: thread (d, j) of a block sums CTAs j, j + 64, ...
// for one of its 16 values, then the 64 sums are added as a tree.
__global__ void __launch_bounds__(1024) dw_sum_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                      float* __restrict__ dwk, int n_part, int D) {
  __shared__ float red[64][17];
  const int i = threadIdx.x & 15, d = blockIdx.x * 16 + i, j = threadIdx.x >> 4;  // D is a multiple of 16
  float s = 0.f;
#pragma unroll 8
  for (int c = j; c < n_part; c += 64) s += __ldg(part + static_cast<int64_t>(c) * 2 * D + d);
  red[j][i] = s;
  __syncthreads();
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) {
    if (j < w) red[j][i] += red[j + w][i];
    __syncthreads();
  }
  if (j == 0) (d < D ? dwq : dwk)[d < D ? d : d - D] = red[0][i];
}

int lanes_of(int D) { return D <= 64 ? 4 : D <= 128 ? 8 : 16; }

constexpr int kMaxPart = 2048;  // CTAs of a backward pass with norms

template <typename T, int L>
int launch_fwd_l(const Args& p, bool norm, bool axes, int w_dtype, float sign, cudaStream_t s) {
  const int64_t tiles = (p.n_tok + kThreads / L - 1) / (kThreads / L);
  // Few tokens: the heads of a token over several CTAs, until there are four for every SM. At 2,000 tokens
  // of 12 / 2 heads that takes 4.1 us, up to 6, 8 and 12 for every SM 5.6, 5.7 and 7.2 (the angles are
  // computed again in each); at 10,000 of 16 / 4 heads of 64 12.9 against 14.0, 12.7 and 12.4.
  const int heads = p.hq + p.hk;
  int64_t groups = 4 * static_cast<int64_t>(sm_count()) / tiles;
  groups = groups < 1 ? 1 : groups > heads ? heads : groups;
  const int per_group = static_cast<int>((heads + groups - 1) / groups);
  const dim3 grid(static_cast<unsigned>(tiles), (heads + per_group - 1) / per_group);
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(p, w_dtype, per_group, sign); };
  const bool lora = p.ql.ptr != nullptr;
  auto pick = [&](auto part) {
    constexpr bool P = decltype(part)::value;
    if (norm) {
      if (axes) lora ? go(fwd_kernel<T, L, true, true, true, P>) : go(fwd_kernel<T, L, true, true, false, P>);
      else lora ? go(fwd_kernel<T, L, true, false, true, P>) : go(fwd_kernel<T, L, true, false, false, P>);
    } else {
      lora ? go(fwd_kernel<T, L, false, true, true, P>) : go(fwd_kernel<T, L, false, true, false, P>);
    }
  };
  if (p.R < p.D) pick(std::true_type()); else pick(std::false_type());
  return check_launch("head_rope_fwd");
}

template <typename T, int L, bool AXES, bool LORA, bool PART>
int launch_bwd_k(const Args& p, int w_dtype, int* n_part, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = norm_bwd_kernel<T, L, AXES, LORA, PART>;
  if (int rc = ensure_dyn_smem(kernel, bwd_smem<L, LORA>(), done, "head_rope_bwd")) return rc;
  const int64_t rows = (p.n_tok + 32 / L - 1) / (32 / L) * (p.hq + p.hk);
  // All CTAs that run at once, however few rows each warp then has: 830 tokens of 12 / 2 heads take 8.1 us, with
  // at least 6 rows a warp 8.5, with 12 10.8; 5,050 of 3 / 3 heads 12.1, 11.6, 13.7.
  int64_t ctas = static_cast<int64_t>(sm_count()) * (LORA ? 3 : 4);
  if (ctas > kMaxPart) ctas = kMaxPart;
  const int64_t warps = ctas * (kThreads / 32), per_warp = (rows + warps - 1) / warps;
  const int64_t used = (rows + per_warp - 1) / per_warp;
  const int grid = static_cast<int>((used + kThreads / 32 - 1) / (kThreads / 32));
  *n_part = grid;
  kernel<<<grid, kThreads, bwd_smem<L, LORA>(), s>>>(p, w_dtype, rows, per_warp);
  return check_launch("head_rope_bwd");
}

template <typename T, int L>
int launch_bwd_l(const Args& p, bool axes, int w_dtype, int* n_part, cudaStream_t s) {
  const bool lora = p.ql.ptr != nullptr;
  auto pick = [&](auto part) {
    constexpr bool P = decltype(part)::value;
    if (axes) return lora ? launch_bwd_k<T, L, true, true, P>(p, w_dtype, n_part, s)
                          : launch_bwd_k<T, L, true, false, P>(p, w_dtype, n_part, s);
    return lora ? launch_bwd_k<T, L, false, true, P>(p, w_dtype, n_part, s)
                : launch_bwd_k<T, L, false, false, P>(p, w_dtype, n_part, s);
  };
  return p.R < p.D ? pick(std::true_type()) : pick(std::false_type());
}

template <typename T>
int launch_fwd(const Args& p, bool norm, bool axes, int w_dtype, float sign, cudaStream_t s) {
  switch (lanes_of(p.D)) {
    case 4: return launch_fwd_l<T, 4>(p, norm, axes, w_dtype, sign, s);
    case 8: return launch_fwd_l<T, 8>(p, norm, axes, w_dtype, sign, s);
    default: return launch_fwd_l<T, 16>(p, norm, axes, w_dtype, sign, s);
  }
}
template <typename T>
int launch_bwd(const Args& p, bool axes, int w_dtype, int* n_part, cudaStream_t s) {
  switch (lanes_of(p.D)) {
    case 4: return launch_bwd_l<T, 4>(p, axes, w_dtype, n_part, s);
    case 8: return launch_bwd_l<T, 8>(p, axes, w_dtype, n_part, s);
    default: return launch_bwd_l<T, 16>(p, axes, w_dtype, n_part, s);
  }
}

bool view_ok(const void* ptr, int64_t ts, int64_t hs) { return ptr && aligned16(ptr) && ts % 8 == 0 && hs % 8 == 0; }

int check(const char* what, const Args& p, bool norm, bool bwd, int w_dtype, int dtype) {
  if (p.n_tok < 0 || p.n_tok > (int64_t(1) << 31) - 1 || p.hq <= 0 || p.hk <= 0 || p.D <= 0 || p.D % 16 != 0 ||
      p.D > 256 || p.R <= 0 || p.R % 16 != 0 || p.R > p.D)
    return set_error(DECIK_ERR_INVALID, "%s: T=%lld, heads %d/%d, head_dim %d, rotary_dim %d (multiples of 16, "
                     "rotary_dim <= head_dim <= 256)", what, (long long)p.n_tok, p.hq, p.hk, p.D, p.R);
  if (dtype != DECIK_F16 && dtype != DECIK_BF16)
    return set_error(DECIK_ERR_INVALID, "%s: dtype %d is not F16/BF16", what, dtype);
  if ((p.wq == nullptr) != (p.wk == nullptr))
    return set_error(DECIK_ERR_INVALID, "%s: norm weights for both queries and keys, or for neither", what);
  if (norm && ((w_dtype != DECIK_F32 && w_dtype != DECIK_F16 && w_dtype != DECIK_BF16) || !(p.eps >= 0.f)))
    return set_error(DECIK_ERR_INVALID, "%s: norm weights of dtype %d (F32, F16 or BF16), eps %g", what, w_dtype,
                     static_cast<double>(p.eps));
  if (p.n_tok == 0) return DECIK_OK;
  bool ok = view_ok(p.oq.ptr, p.oq.tok_stride, p.oq.head_stride) && view_ok(p.ok.ptr, p.ok.tok_stride, p.ok.head_stride);
  if (!bwd || norm)
    ok = ok && view_ok(p.q.ptr, p.q.tok_stride, p.q.head_stride) && view_ok(p.k.ptr, p.k.tok_stride, p.k.head_stride) &&
         (!p.ql.ptr || view_ok(p.ql.ptr, p.ql.tok_stride, p.ql.head_stride));
  if (bwd)
    ok = ok && view_ok(p.gq.ptr, p.gq.tok_stride, p.gq.head_stride) &&
         view_ok(p.gk.ptr, p.gk.tok_stride, p.gk.head_stride);
  if (!ok) return set_error(DECIK_ERR_INVALID, "%s: a view is NULL, or its pointer or strides are not 16-byte aligned", what);
  if (norm && (!aligned_to(p.wq, dtype_bytes(w_dtype)) || !aligned_to(p.wk, dtype_bytes(w_dtype))))
    return set_error(DECIK_ERR_INVALID, "%s: a norm weight is not aligned to its values", what);
  return DECIK_OK;
}

int set_tables(const char* what, Args& p, const float* cos, const float* sin) {
  if (p.n_tok != 0 && (!cos || !sin || !aligned16(cos) || !aligned16(sin)))
    return set_error(DECIK_ERR_INVALID, "%s: cos / sin NULL or not 16-byte aligned", what);
  p.ang.cos = cos;
  p.ang.sin = sin;
  return DECIK_OK;
}

int set_axes(const char* what, Args& p, const void* positions, int pos_dtype, int64_t ld_pos, int n_axes,
             const float* inv_freq, const uint8_t* axis_of) {
  if (n_axes < 1 || n_axes > 4 || (pos_dtype != 0 && pos_dtype != 1))
    return set_error(DECIK_ERR_INVALID, "%s: %d axes (1 to 4), position dtype %d (0 = int64, 1 = int32)", what, n_axes,
                     pos_dtype);
  if (!axis_of || (p.n_tok != 0 && (!positions || !inv_freq)) || (n_axes > 1 && ld_pos < p.n_tok))
    return set_error(DECIK_ERR_INVALID, "%s: null pointer, or rows of positions shorter than the tokens", what);
  if (p.n_tok != 0 && !aligned_to(positions, pos_dtype == 1 ? 4 : 8))
    return set_error(DECIK_ERR_INVALID, "%s: positions are not aligned to their values", what);
  if (p.n_tok != 0 && !aligned16(inv_freq))  // load_angles reads it in 16-byte pieces
    return set_error(DECIK_ERR_INVALID, "%s: inv_freq is not 16-byte aligned", what);
  p.ang.pos = positions;
  p.ang.pos32 = pos_dtype;
  p.ang.n_axes = n_axes;
  p.ang.ld_pos = ld_pos;
  p.ang.inv_freq = inv_freq;
  for (int j = 0; j < 8; ++j) p.ang.axis[j] = 0;
  for (int j = 0; j < p.R / 2; ++j) {
    if (axis_of[j] >= n_axes)
      return set_error(DECIK_ERR_INVALID, "%s: frequency %d has axis %d of %d", what, j, axis_of[j], n_axes);
    p.ang.axis[j >> 4] |= static_cast<uint32_t>(axis_of[j]) << (2 * (j & 15));
  }
  return DECIK_OK;
}

int run_fwd(const char* what, const Args& p, bool axes, int w_dtype, int dtype, cudaStream_t s) {
  if (int rc = check(what, p, p.wq != nullptr, false, w_dtype, dtype)) return rc;
  if (p.n_tok == 0) return DECIK_OK;
  return DECIK_DISPATCH_16(dtype, [&] { return launch_fwd<T>(p, p.wq != nullptr, axes, w_dtype, 1.f, s); });
}

int run_bwd(const char* what, Args p, bool axes, int w_dtype, float* dwq, float* dwk, void* workspace, int dtype,
            cudaStream_t s) {
  const bool norm = p.wq != nullptr;
  if (int rc = check(what, p, norm, true, w_dtype, dtype)) return rc;
  if (norm && (!dwq || !dwk)) return set_error(DECIK_ERR_INVALID, "%s: dq_weight or dk_weight NULL", what);
  if (norm && (!aligned_to(dwq, 4) || !aligned_to(dwk, 4)))
    return set_error(DECIK_ERR_INVALID, "%s: dq_weight or dk_weight is not aligned to its values", what);
  if (p.n_tok == 0) {
    cudaError_t e = cudaSuccess;
    if (norm) e = cudaMemsetAsync(dwq, 0, sizeof(float) * p.D, s);
    if (norm && e == cudaSuccess) e = cudaMemsetAsync(dwk, 0, sizeof(float) * p.D, s);
    return e == cudaSuccess ? DECIK_OK : set_error(DECIK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  if (norm && (!workspace || !aligned16(workspace)))
    return set_error(DECIK_ERR_INVALID, "%s: workspace NULL or not 16-byte aligned", what);
  if (!norm) {  // the rotation back, from the gradients
    p.q = p.gq;
    p.k = p.gk;
    p.ql = {};
    return DECIK_DISPATCH_16(dtype, [&] { return launch_fwd<T>(p, false, axes, w_dtype, -1.f, s); });
  }
  p.part = static_cast<float*>(workspace);
  int n_part = 0;
  if (int rc = DECIK_DISPATCH_16(dtype, [&] { return launch_bwd<T>(p, axes, w_dtype, &n_part, s); })) return rc;
  dw_sum_kernel<<<2 * p.D / 16, 1024, 0, s>>>(p.part, dwq, dwk, n_part, p.D);
  return check_launch(what);
}

}  // namespace
}  // namespace headrope
}  // namespace decik

extern "C" int decik_qk_norm_rope_fwd(decik_tensor3 q, decik_tensor3 q_lora, decik_tensor3 k, const void* q_weight,
                                      const void* k_weight, int w_dtype, float eps, const float* cos, const float* sin,
                                      decik_tensor3_mut q_out, decik_tensor3_mut k_out, int64_t n_tok, int n_heads,
                                      int n_kv, int head_dim, int rotary_dim, int dtype, void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, {}, {}, q_out, k_out, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (!q_weight || !k_weight) return decik::set_error(DECIK_ERR_INVALID, "qk_norm_rope_fwd: NULL norm weight");
  if (int rc = set_tables("qk_norm_rope_fwd", p, cos, sin)) return rc;
  return run_fwd("qk_norm_rope_fwd", p, false, w_dtype, dtype, decik::as_stream(stream));
}

extern "C" int decik_rope_axes_fwd(decik_tensor3 q, decik_tensor3 q_lora, decik_tensor3 k, const void* q_weight,
                                   const void* k_weight, int w_dtype, float eps, const void* positions, int pos_dtype,
                                   int64_t ld_pos, int n_axes, const float* inv_freq, const uint8_t* axis_of,
                                   decik_tensor3_mut q_out, decik_tensor3_mut k_out, int64_t n_tok, int n_heads,
                                   int n_kv, int head_dim, int rotary_dim, int dtype, void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, {}, {}, q_out, k_out, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (int rc = check("rope_axes_fwd", p, q_weight != nullptr, false, w_dtype, dtype)) return rc;  // R before axis_of[R / 2]
  if (int rc = set_axes("rope_axes_fwd", p, positions, pos_dtype, ld_pos, n_axes, inv_freq, axis_of)) return rc;
  return run_fwd("rope_axes_fwd", p, true, w_dtype, dtype, decik::as_stream(stream));
}

extern "C" int64_t decik_qk_norm_rope_bwd_workspace(int head_dim) {
  return head_dim <= 0 ? 0 : static_cast<int64_t>(decik::headrope::kMaxPart) * 2 * head_dim * sizeof(float);
}

extern "C" int decik_qk_norm_rope_bwd(decik_tensor3 grad_q, decik_tensor3 grad_k, decik_tensor3 q, decik_tensor3 q_lora,
                                      decik_tensor3 k, const void* q_weight, const void* k_weight, int w_dtype,
                                      float eps, const float* cos, const float* sin, decik_tensor3_mut dq,
                                      decik_tensor3_mut dk, float* dq_weight, float* dk_weight, int64_t n_tok,
                                      int n_heads, int n_kv, int head_dim, int rotary_dim, int dtype, void* workspace,
                                      void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, grad_q, grad_k, dq, dk, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (!q_weight || !k_weight) return decik::set_error(DECIK_ERR_INVALID, "qk_norm_rope_bwd: NULL norm weight");
  if (int rc = set_tables("qk_norm_rope_bwd", p, cos, sin)) return rc;
  return run_bwd("qk_norm_rope_bwd", p, false, w_dtype, dq_weight, dk_weight, workspace, dtype,
                 decik::as_stream(stream));
}

extern "C" int decik_rope_axes_bwd(decik_tensor3 grad_q, decik_tensor3 grad_k, decik_tensor3 q, decik_tensor3 q_lora,
                                   decik_tensor3 k, const void* q_weight, const void* k_weight, int w_dtype, float eps,
                                   const void* positions, int pos_dtype, int64_t ld_pos, int n_axes,
                                   const float* inv_freq, const uint8_t* axis_of, decik_tensor3_mut dq,
                                   decik_tensor3_mut dk, float* dq_weight, float* dk_weight, int64_t n_tok,
                                   int n_heads, int n_kv, int head_dim, int rotary_dim, int dtype, void* workspace,
                                   void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, grad_q, grad_k, dq, dk, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (int rc = check("rope_axes_bwd", p, q_weight != nullptr, true, w_dtype, dtype)) return rc;
  if (int rc = set_axes("rope_axes_bwd", p, positions, pos_dtype, ld_pos, n_axes, inv_freq, axis_of)) return rc;
  return run_bwd("rope_axes_bwd", p, true, w_dtype, dq_weight, dk_weight, workspace, dtype,
                 decik::as_stream(stream));
}
