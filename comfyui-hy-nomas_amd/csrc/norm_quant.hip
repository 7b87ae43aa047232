// Residual addition, RMS norm and 8-bit quantization of a decoder layer's input in one kernel: the pre-norm in front of
// an fp8 or int8 linear (the decoder's RMSNorm, hy_nomas/pixelumm.py:246-259, then kernels.py:22-54 on its result).
//
//   h = T(x + r)                                  (the layer's new residual stream, in the tensors' type T)
//   y = h / sqrt(mean(h^2) + eps) * w             (fp32, not rounded to T)
//   s = scale of max |y| over a group             (int8: peak / 127, 1 for an all-zero group; e4m3: max(peak, 1e-12) / 448)
//   q = code of y / s
//
// One pass, bound by memory: a row is read once into registers by WPR waves (one, or four for long rows and for calls of few
// rows), 8 values a lane and chunk, with non-temporal accesses (plain ones were 3 to 7 % slower over rows that no cache holds);
// 35200 rows of 4096 values with a residual 166 us in bf16, 6.1 TB/s of a copy's 6.6; 164 in fp16; 360 in fp32,
// 5.2 TB/s.  The codes do not wait for the row's statistics:
// with t = h w the quotient y / s is t / (max |t| / 127), so each group's quotients come from the group alone and only the scale,
// max |t| rstd / 127, needs rstd.  Groups
// whose products lie outside [2^-80, 2^100], where t or its reciprocal could leave fp32's normal range (all-zero and
// non-finite ones among them), and e4m3 groups under the 1e-12 floor take the formula as it stands instead.
#include "quant_codes.h"

namespace hn {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
  const void *x, *r, *w;
  int64_t ldx, ldr, ldh, ldq, lds, M, D;
  void* h;
  uint8_t* q;
  float* s;
  float eps;
  int rounding, w_f32;
};

template <int DT>
struct Eight {  // 8 consecutive values of a row
  static constexpr int kBytes = DT == HN_DTYPE_F32 ? 32 : 16;
  uint4 v[kBytes / 16];
  __device__ __forceinline__ void load_nt(const void* row, int c) {
    const char* p = (const char*)row + (int64_t)c * kBytes;
#pragma unroll
    for (int i = 0; i < kBytes / 16; i++) v[i] = ld_nt16(p + 16 * i);
  }
  __device__ __forceinline__ void load(const void* row, int c) {
    const uint4* p = (const uint4*)((const char*)row + (int64_t)c * kBytes);
#pragma unroll
    for (int i = 0; i < kBytes / 16; i++) v[i] = p[i];
  }
  __device__ __forceinline__ void store_nt(void* row, int c) const {
    char* p = (char*)row + (int64_t)c * kBytes;
#pragma unroll
    for (int i = 0; i < kBytes / 16; i++) st_nt16(p + 16 * i, v[i]);
  }
  __device__ __forceinline__ void widen(float* f) const {
    if constexpr (DT == HN_DTYPE_F32) {
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = __uint_as_float(w[i]);
    } else {
      In<DT>::widen8(v[0], f);
    }
  }
  // f rounded to the type (a NaN stays one), in both forms
  __device__ __forceinline__ void narrow(float* f) {
    if constexpr (DT == HN_DTYPE_F32) {
      v[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      v[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (DT == HN_DTYPE_F16) {  // the fp32 sum first (no mixed-precision add straight to fp16)
          asm volatile("" : "+v"(f[2 * i]));
          asm volatile("" : "+v"(f[2 * i + 1]));
          w[i] = f32_to_f16_bits(f[2 * i]) | (f32_to_f16_bits(f[2 * i + 1]) << 16);
        } else {
          w[i] = bf16x2_finite(f[2 * i], f[2 * i + 1]);
        }
      }
      v[0] = make_uint4(w[0], w[1], w[2], w[3]);
      widen(f);
    }
  }
};

__device__ __forceinline__ void weight8(const NormArgs& a, int c, float* w, Eight<HN_DTYPE_F32>*) {
  Eight<HN_DTYPE_F32> e;
  e.load(a.w, c);
  e.widen(w);
}
template <int DT>
__device__ __forceinline__ void weight8(const NormArgs& a, int c, float* w, Eight<DT>*) {
  if (a.w_f32) return weight8(a, c, w, (Eight<HN_DTYPE_F32>*)nullptr);
  Eight<DT> e;
  e.load(a.w, c);
  e.widen(w);
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // ordered as |v|, NaN on top

__device__ __forceinline__ uint32_t row16_max(uint32_t u) {
  u = max(u, dpp_u<0xB1>(u));
  u = max(u, dpp_u<0x4E>(u));
  u = max(u, dpp_u<0x141>(u));
  return max(u, dpp_u<0x140>(u));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t u) {
  u = row16_max(u);
  u = max(u, dpp_u<0x142, 0xa>(u));
  u = max(u, dpp_u<0x143, 0xc>(u));
  return (uint32_t)__builtin_amdgcn_readlane((int)u, 63);
}

// The reciprocal of a group's peak |t|, which is given by its magnitude bits, and the group's scale; ok: whether they may be used.
template <int KIND>
struct GroupFactor {
  float rcp, scale;
  bool ok;
  __device__ __forceinline__ GroupFactor(uint32_t peak_bits, float rstd) {
    const float top = KIND == HN_KIND_FP8 ? 448.0f : 127.0f;
    const float peak = __uint_as_float(peak_bits);
    const float r0 = __builtin_amdgcn_rcpf(peak);
    rcp = __builtin_fmaf(__builtin_fmaf(-r0, peak, 1.0f), r0, r0);
    const float y = peak * rstd;
    scale = div_by_const(y, top, 1.0f / top);
    // [2^-80, 2^100] on the bits, so that a NaN is outside; y a normal number
    ok = peak_bits - 0x17800000u <= 0x71800000u - 0x17800000u && y >= (KIND == HN_KIND_FP8 ? 1e-12f : 0x1p-100f) && y < 0x1p100f;
  }
};

// The formula as it stands, for a group whose peak |y| is given by its magnitude bits.
template <int KIND>
__device__ __forceinline__ float plain_scale(uint32_t peak_bits) {
  const float peak = __uint_as_float(peak_bits);
  if (peak != peak) return peak;  // a NaN in the group shows in its scale
  return KIND == HN_KIND_FP8 ? fp8_scale(peak) : int8_scale(peak);
}

template <int KIND>
__device__ __forceinline__ uint2 plain_codes(const float* y, float scale, int rounding) {
  if constexpr (KIND == HN_KIND_FP8) return encode8<KIND, HN_ROUND_HALF_AWAY, false>(y, scale);
  else
    return rounding == HN_ROUND_HALF_EVEN ? encode8<KIND, HN_ROUND_HALF_EVEN, false>(y, scale)
                                          : encode8<KIND, HN_ROUND_HALF_AWAY, false>(y, scale);
}

// The codes of z = t top / peak rounded once: int8 by `rounding`, e4m3 to even.
template <int KIND, bool STICKY>
__device__ __forceinline__ uint2 quotient_codes(const float* z, int rounding) {
  if constexpr (KIND == HN_KIND_FP8) {
    return make_uint2(e4m3_pack4_hw(z[0], z[1], z[2], z[3]), e4m3_pack4_hw(z[4], z[5], z[6], z[7]));
  } else {
    int c[8];
#pragma unroll
    for (int j = 0; j < 8; j++)  // STICKY: half away by the float below 0.5, whose sum with a value under a half stays under
      c[j] = rounding == HN_ROUND_HALF_EVEN ? rne_code_bits(z[j])
             : STICKY                       ? (int)(z[j] + __builtin_copysignf(0x1.fffffep-2f, z[j]))
                                            : round_half_away_i8_inrange(z[j]);
    return make_uint2(pack4_i8(c[0], c[1], c[2], c[3]), pack4_i8(c[4], c[5], c[6], c[7]));
  }
}

// t top / peak with the quotient's rounding error mended: where it lies halfway between two codes, as 1 in 2300 does with
// bf16 values and weights, it is formed exactly and goes to the code that the rounding says.  (A product with top / peak alone
// gave half of those to the other neighbour.)  A bf16 product h w has 16 bits, so t top is exact, and quotients that are no
// ties lie further from one than fp32's rounding reaches.
//
// WIDE, fp16 values: t has up to 22 bits and t top up to 29, so a quotient may lie within fp32's rounding of a tie.  z is within
// 2^-23 of the quotient, relatively; a lane with a z within four steps of a tie (for e4m3 also one of its subnormals) forms
// its quotients with the product's low part in the remainder.  The last remainder e then tells on which side the
// quotient lies, and z becomes its odd neighbour (the quotient itself where e is 0), which no boundary of codes is: the rounding to
// a code sees what a quotient of unlimited precision would show it.  (35200 rows of 1024 take
// 42.9 us, 777 of 2560 5.25; 43.9 and 5.75 with every lane doing so, 41.9 and 5.1 with ties left to chance.)
template <int KIND, bool WIDE>
__device__ __forceinline__ uint2 fast_codes(const float* t, float rcp, float peak, int rounding) {
  constexpr float top = KIND == HN_KIND_FP8 ? 448.0f : 127.0f;
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float n = t[j] * top, q = n * rcp;
    z[j] = __builtin_fmaf(__builtin_fmaf(-q, peak, n), rcp, q);
  }
  if constexpr (!WIDE) return quotient_codes<KIND, false>(z, rounding);
  uint2 codes;
  bool near;
  if constexpr (KIND == HN_KIND_FP8) {
    codes = quotient_codes<KIND, false>(z, rounding);
    uint32_t above = ~0u;
    float least = 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {  // a tie: the 20 bits below e4m3's mantissa are 0x80000
      above = min(above, (__float_as_uint(z[j]) - 0x7fffcu) & 0xfffffu);
      least = __builtin_fminf(least, __builtin_fabsf(z[j]));
    }
    near = above <= 8u || least < 0x1p-6f;
  } else {
    float off = 0.0f;
    int c[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {  // away from ties both roundings are the nearest code
      const float r = __builtin_rintf(z[j]);
      off = __builtin_fmaxf(off, __builtin_fabsf(z[j] - r));
      c[j] = (int)r;
    }
    codes = make_uint2(pack4_i8(c[0], c[1], c[2], c[3]), pack4_i8(c[4], c[5], c[6], c[7]));
    near = off >= 0.5f - 0x1p-15f;  // (four steps of a z next to 127)
  }
  if (__builtin_expect(near, 0)) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float n = t[j] * top, q = n * rcp, lo = __builtin_fmaf(t[j], top, -n);
      const float about = __builtin_fmaf(__builtin_fmaf(-q, peak, n) + lo, rcp, q);
      const float e = __builtin_fmaf(-about, peak, n) + lo;
      const uint32_t bits = __float_as_uint(about);
      const uint32_t below = (uint32_t)((int)(bits ^ __float_as_uint(e)) >> 31);  // -1 where the quotient is nearer to zero
      z[j] = __uint_as_float(e == 0.0f ? bits : (bits + below) | 1u);
    }
    codes = quotient_codes<KIND, true>(z, rounding);
  }
  return codes;
}

// WPR waves a row, CPL chunks of 8 values a lane; PT: one scale a row.
template <int DT, int KIND, bool PT, int WPR, int CPL>
__global__ __launch_bounds__(kThreads) void rms_norm_quant_kernel(const NormArgs a) {
  __shared__ float2 part[WPR == 1 ? 1 : WPR];
  constexpr int kRows = kThreads / 64 / WPR;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * kRows + (WPR == 1 ? wave : 0);
  if (row >= a.M) return;  // whole waves, and with WPR > 1 never
  const int first = WPR == 1 ? lane : (int)threadIdx.x;  // chunk i of this lane: first + 64 WPR i
  constexpr int kStep = 64 * WPR;
  const int chunks = (int)(a.D / 8);
  constexpr int eb = DT == HN_DTYPE_F32 ? 4 : 2;
  const char* xr = (const char*)a.x + row * a.ldx * eb;
  const char* rr = (const char*)a.r + row * a.ldr * eb;
  char* hr = (char*)a.h + row * a.ldh * eb;
  Eight<DT> xv[CPL], rv[CPL];
#pragma unroll
  for (int i = 0; i < CPL; i++)
    if (first + kStep * i < chunks) xv[i].load_nt(xr, first + kStep * i);
  if (a.r) {
#pragma unroll
    for (int i = 0; i < CPL; i++)
      if (first + kStep * i < chunks) rv[i].load_nt(rr, first + kStep * i);
  }
  float t[CPL][8], sq = 0.0f;
  uint32_t peak[CPL];
#pragma unroll
  for (int i = 0; i < CPL; i++) {
    peak[i] = 0;
    if (first + kStep * i < chunks) {
      float w[8];
      xv[i].widen(t[i]);
      if (a.r) {
        float r[8];
        rv[i].widen(r);
#pragma unroll
        for (int j = 0; j < 8; j++) t[i][j] += r[j];
        xv[i].narrow(t[i]);
        xv[i].store_nt(hr, first + kStep * i);
      }
      weight8(a, first + kStep * i, w, (Eight<DT>*)nullptr);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        sq = __builtin_fmaf(t[i][j], t[i][j], sq);
        t[i][j] *= w[j];
        peak[i] = max(peak[i], magnitude(t[i][j]));
      }
    }
  }
  uint32_t top = 0;  // PT: of the row
  if constexpr (PT) {
#pragma unroll
    for (int i = 0; i < CPL; i++) top = max(top, peak[i]);
    top = wave_max_u(top);
  }
  sq = wave_sum_dpp(sq);
  if constexpr (WPR > 1) {
    if (lane == 0) part[wave] = make_float2(sq, __uint_as_float(top));
    __syncthreads();
    sq = 0.0f;
    top = 0;
#pragma unroll
    for (int k = 0; k < WPR; k++) {
      sq += part[k].x;
      top = max(top, __float_as_uint(part[k].y));
    }
  }
  const float rstd = rsqrt_refined(sq / (float)a.D + a.eps);
  uint8_t* qr = a.q + row * a.ldq;
  float* sr = a.s + row * a.lds;
  // chunk i's channels again, as t = h w and as y = h rstd w, for groups the factors are not for
  auto formula = [&](int i, float* t, float* y) {
    Eight<DT> e;
    float w[8];
    e.load(a.r ? (const char*)hr : xr, first + kStep * i);
    e.widen(y);
    weight8(a, first + kStep * i, w, (Eight<DT>*)nullptr);
    uint32_t p = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      t[j] = y[j] * w[j];
      y[j] = y[j] * rstd * w[j];
      p = max(p, magnitude(y[j]));
    }
    return p;
  };
  if constexpr (PT) {
    const GroupFactor<KIND> g(top, rstd);
    if (__builtin_expect(g.ok, 1)) {  // the same in the whole row
#pragma unroll
      for (int i = 0; i < CPL; i++)
        if (first + kStep * i < chunks) st_nt8(qr + (first + kStep * i) * 8, fast_codes<KIND, DT == HN_DTYPE_F16>(t[i], g.rcp, __uint_as_float(top), a.rounding));
      if (first == 0) sr[0] = g.scale;
      return;
    }
    top = 0;
#pragma unroll 1
    for (int c = first, i = 0; c < chunks; c += kStep, i++) {
      float again[8], y[8];
      top = max(top, formula(i, again, y));
    }
    top = wave_max_u(top);
    if constexpr (WPR > 1) {
      __syncthreads();
      if (lane == 0) part[wave].y = __uint_as_float(top);
      __syncthreads();
      for (int k = 0; k < WPR; k++) top = max(top, __float_as_uint(part[k].y));
    }
    const float sc = plain_scale<KIND>(top);
#pragma unroll 1
    for (int c = first, i = 0; c < chunks; c += kStep, i++) {
      float again[8], y[8];
      formula(i, again, y);
      st_nt8(qr + c * 8, plain_codes<KIND>(y, sc, a.rounding));
    }
    if (first == 0) sr[0] = sc;
  } else {
    // 16 lanes hold a group of 128 channels.  Lane k of the 16 forms chunk k's factor and scale, and the others read the
    // factor from it; lanes k >= CPL repeat chunk 0's.
    static_assert(CPL <= 16, "a lane of the 16 for each chunk");
    const int k = lane & 15;
#pragma unroll
    for (int i = 0; i < CPL; i++) peak[i] = row16_max(peak[i]);
    uint32_t mine = peak[0];
    int at = first;  // its group's chunk in this lane
#pragma unroll
    for (int i = 1; i < CPL; i++)
      if (k == i) {
        mine = peak[i];
        at = first + kStep * i;
      }
    const bool has = at < chunks;  // (a group's 16 chunks all lie in the row or none does)
    const GroupFactor<KIND> g(mine, rstd);
    if (__builtin_expect(__all(g.ok || !has), 1)) {
#pragma unroll
      for (int i = 0; i < CPL; i++) {
        const float f = row_bcast(g.rcp, i);
        if (first + kStep * i < chunks) st_nt8(qr + (first + kStep * i) * 8, fast_codes<KIND, DT == HN_DTYPE_F16>(t[i], f, __uint_as_float(peak[i]), a.rounding));
      }
      if (k < CPL && has) sr[at / 16] = g.scale;
      return;
    }
    // Some group of the wave has no factor (pruned channels, say): it alone takes the formula, so that a group's codes never
    // depend on what lies in another.  (The products are formed again: kept for here, they slowed the path above by 2 to 4 %.)
#pragma unroll 1
    for (int c = first, i = 0; c < chunks; c += kStep, i++) {
      float again[8], y[8];
      const uint32_t peak_y = row16_max(formula(i, again, y));
      uint32_t p = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) p = max(p, magnitude(again[j]));
      p = row16_max(p);
      const GroupFactor<KIND> own(p, rstd);
      if (own.ok) {  // the same in the group's 16 lanes
        st_nt8(qr + c * 8, fast_codes<KIND, DT == HN_DTYPE_F16>(again, own.rcp, __uint_as_float(p), a.rounding));
        if (k == 0) sr[c / 16] = own.scale;
      } else {
        const float sc = plain_scale<KIND>(peak_y);
        st_nt8(qr + c * 8, plain_codes<KIND>(y, sc, a.rounding));
        if (k == 0) sr[c / 16] = sc;
      }
    }
  }
}

template <int DT, int KIND, bool PT, int WPR>
int launch_norm(const NormArgs& a, hipStream_t st) {
  const int64_t cpl = (a.D / 8 + 64 * WPR - 1) / (64 * WPR);
  constexpr int rows = kThreads / 64 / WPR;
  const dim3 grid((unsigned)((a.M + rows - 1) / rows)), block(kThreads);
#define HN_NORM_CASE(N)                                                                       \
  if (cpl <= N) {                                                                             \
    hipLaunchKernelGGL((rms_norm_quant_kernel<DT, KIND, PT, WPR, N>), grid, block, 0, st, a); \
    return HN_LAUNCH_CHECK("rms_norm_quant_kernel");                                          \
  }
  HN_NORM_CASE(1) HN_NORM_CASE(2) HN_NORM_CASE(4)
  if constexpr (WPR > 1) {  // (one wave takes rows of up to 2048 values)
    HN_NORM_CASE(6) HN_NORM_CASE(8)
  }
#undef HN_NORM_CASE
  set_error("hn_rms_norm_quant: D=%lld out of range", (long long)a.D);
  return HN_ERR_UNSUPPORTED;
}

template <int DT>
int dispatch_norm(const NormArgs& a, int kind, bool per_token, hipStream_t st) {
  // A wave a row where rows fill the chip and are short, else four: 35200 rows of 1024 values 42.6 against 50.2 us, of 4096
  // 173.7 against 164.3, 26400 of 2048 64.0 against 62.4, 1500 of 2048 5.9 against 4.7.
  const bool one = a.D <= 2048 && a.M >= 8 * cu_count();
#define HN_NORM_WPR(K, PT) return one ? launch_norm<DT, K, PT, 1>(a, st) : launch_norm<DT, K, PT, 4>(a, st)
  if (kind == HN_KIND_FP8) {
    if (per_token) HN_NORM_WPR(HN_KIND_FP8, true);
    HN_NORM_WPR(HN_KIND_FP8, false);
  }
  if (per_token) HN_NORM_WPR(HN_KIND_INT8, true);
  HN_NORM_WPR(HN_KIND_INT8, false);
#undef HN_NORM_WPR
}

}  // namespace
}  // namespace hn

extern "C" int hn_rms_norm_quant(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                 int weight_dtype, int dtype, int64_t M, int64_t D, float eps, int kind, int rounding,
                                 int64_t group, void* h, int64_t ldh, void* q, int64_t ldq, float* s, int64_t lds,
                                 void* stream) {
  using namespace hn;
  HN_REQUIRE(dtype >= HN_DTYPE_BF16 && dtype <= HN_DTYPE_F32, "hn_rms_norm_quant: bad dtype %d", dtype);
  HN_REQUIRE(weight_dtype == dtype || weight_dtype == HN_DTYPE_F32, "hn_rms_norm_quant: weight of x's type or fp32, got %d",
             weight_dtype);
  HN_REQUIRE(M >= 0 && M <= 0x7fffffff && D > 0 && D % 128 == 0 && D <= 16384,
             "hn_rms_norm_quant: M=%lld, D=%lld (a multiple of 128 up to 16384)", (long long)M, (long long)D);
  HN_REQUIRE(group == 128 || group == D, "hn_rms_norm_quant: group must be 128 or D (got %lld)", (long long)group);
  HN_REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8, "hn_rms_norm_quant: bad kind %d", kind);
  HN_REQUIRE(rounding == HN_ROUND_HALF_AWAY || rounding == HN_ROUND_HALF_EVEN, "hn_rms_norm_quant: bad rounding %d", rounding);
  HN_REQUIRE(eps > 0.0f && eps < 1e30f, "hn_rms_norm_quant: eps must be positive and finite");
  HN_REQUIRE(x && weight && q && s, "hn_rms_norm_quant: null pointer");
  HN_REQUIRE((residual == nullptr) == (h == nullptr), "hn_rms_norm_quant: a residual and its sum h come together");
  const int64_t per16 = dtype == HN_DTYPE_F32 ? 4 : 8;
  HN_REQUIRE(ldx >= D && ldq >= D && lds >= D / group && (!h || (ldr >= D && ldh >= D)),
             "hn_rms_norm_quant: row strides smaller than the rows");
  HN_REQUIRE(ldx % per16 == 0 && ldq % 8 == 0 && (!h || (ldr % per16 == 0 && ldh % per16 == 0)) && ((uintptr_t)x & 15) == 0 &&
                 ((uintptr_t)residual & 15) == 0 && ((uintptr_t)h & 15) == 0 && ((uintptr_t)weight & 15) == 0 &&
                 ((uintptr_t)q & 7) == 0 && ((uintptr_t)s & 3) == 0,
             "hn_rms_norm_quant: x, residual, h and weight rows must be 16-byte and q rows 8-byte aligned");
  if (M == 0) return HN_OK;
  const NormArgs a{x, residual, weight, ldx, ldr, ldh, ldq, lds, M, D, h, (uint8_t*)q, s, eps, rounding, weight_dtype == HN_DTYPE_F32};
  hipStream_t st = (hipStream_t)stream;
  const bool per_token = group == D && D != 128;
  switch (dtype) {
    case HN_DTYPE_BF16: return dispatch_norm<HN_DTYPE_BF16>(a, kind, per_token, st);
    case HN_DTYPE_F16: return dispatch_norm<HN_DTYPE_F16>(a, kind, per_token, st);
    default: return dispatch_norm<HN_DTYPE_F32>(a, kind, per_token, st);
  }
}
