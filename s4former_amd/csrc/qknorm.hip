// Norm of queries and keys per head with the position rotation in the same pass, and its backward.
//
// One head of one row is x[0:64].  With c_i, s_i (i < 32) the cosines and sines of the row's position and g the gain of its kind
// (query or key; shared by the heads of the kind):
//   r = 1 / sqrt(mean x^2 + eps),  n = x r g,  y_i = n_i c_i - n_{i+32} s_i,  y_{i+32} = n_{i+32} c_i + n_i s_i
// backward, dz = the turn of dy by minus the angle, u = x r:
//   dg = sum dz u  (over rows and the heads of the kind),  dx = r (dz g - u mean(dz g u))
// Everything between the loads and the one rounding of the store is fp32.
//
// Layout: LANES lanes hold a head; a lane has V = 32 / LANES values of the lower and V of the upper half, so that a rotation's pair stays in
// the lane, the mean takes two or three lane exchanges, and one 8-bit group (32 channels: a half) is spread over the same lanes.  Four
// lanes and 16-byte accesses for bf16, eight for fp32; eight also for the backward from x, whose registers then leave room for twice the
// waves (3 x 2,305 rows, 16 + 4 heads, with the join: 13.7 us, with four lanes 15.3; from the checkpoint four are faster by 2 us at 16,400
// rows x 24).  Both passes are bound by HBM; the tables (256 bytes a row) are read per head but come from cache, the heads of a row being
// neighbours in the grid.
//
// Measured at 16,400 rows x 24 heads, calls one behind the other on the same tensors (partly in the last-level cache) / on fresh ones, the
// backward with the join of the gains (4 us; a large copy reaches 4.8 - 5.0 TB/s):
//   bf16  forward 16.6 / 21.9 us (6.1 / 4.6 TB/s), with the checkpoint 21.7 / 28.9, backward from x 27.7 / 33.5, from the checkpoint 25.4 / 32.1
//   fp32  forward 29.6 / 36.6 us (6.8 / 5.5 TB/s), with the checkpoint 34.1 / 41.3, backward from x 51.2 / 59.2, from the checkpoint 39.4 / 46.5
// A call on few rows takes 2.5 - 3.5 us on the GPU, less than its launch costs the host.
#include "actq8.h"
#include "../../include/s4f.h"
#include <algorithm>
#include <cfloat>

namespace {

struct QkArgs {
  const void* x; int64_t ldx;
  const void* dy; int64_t lddy;
  void* y; int64_t ldy;                 // forward: y, backward: dx
  const float *gq, *gk, *cos, *sin;
  int8_t* codes; uint8_t* scales;       // pre-norm checkpoint: written by the forward, read by the backward
  float* part;                          // backward: [blocks][64] partial gain gradients
  float eps;
  uint32_t rows, period;
  int Hq, H;                            // query heads, all heads
  int bq;                               // backward: blocks that take query heads (the others take key heads)
};

// V values of a lane in one access of 8 or 16 bytes
template <typename T, int V> struct __attribute__((aligned(V * sizeof(T)))) Vals { T t[V]; };
template <int V, typename T> __device__ __forceinline__ Vals<T, V> ld_vals(const T* p) { return *reinterpret_cast<const Vals<T, V>*>(p); }
template <typename T, int V> __device__ __forceinline__ void unpack(const Vals<T, V>& c, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (float)c.t[i];
}
template <typename T, int V> __device__ __forceinline__ void st_vals(T* p, const float (&v)[V]) {
  Vals<T, V> c;
#pragma unroll
  for (int i = 0; i < V; ++i) c.t[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Vals<T, V>*>(p) = c;
}
template <int V> struct __attribute__((aligned(V))) Codes { uint32_t w[V / 4]; };           // V codes of a lane
template <int V> __device__ __forceinline__ void ld_f32(const float* p, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(p + i);
    v[i] = q[0]; v[i + 1] = q[1]; v[i + 2] = q[2]; v[i + 3] = q[3];
  }
}

// r of a head whose lanes hold partial sums of squares.  fp32 operands: correctly rounded root and quotient; bf16: the hardware's
// reciprocal root (1 ulp of fp32, 2^-15 of a bf16 step)
template <typename T, int LANES> __device__ __forceinline__ float inv_rms(float sq, float eps) {
  const float m = fmaf(group_sum<LANES>(sq), 1.f / 64.f, eps);
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rsqf(m);
  return 1.f / sqrtf(m);
}

template <typename T, bool NORM, bool ROPE, bool PACK>
__global__ __launch_bounds__(256) void qk_fwd_kernel(const QkArgs a) {
  constexpr int V = 16 / sizeof(T), LANES = 32 / V;
  const int l = threadIdx.x & (LANES - 1);
  const uint32_t it = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (it >= a.rows * (uint32_t)a.H) return;              // (whole groups of lanes)
  const uint32_t row = it / (uint32_t)a.H;
  const int h = (int)(it - row * (uint32_t)a.H);
  const T* xp = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx + h * 64 + l * V;
  float lo[V], hi[V];
  unpack(ld_vals<V>(xp), lo);
  unpack(ld_vals<V>(xp + 32), hi);
  if constexpr (PACK) {
    uint32_t ml = 0, mh = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) { ml = max(ml, mag_bits(lo[e])); mh = max(mh, mag_bits(hi[e])); }
    const uint32_t bl = q8_scale_byte(group_max<LANES>(ml)), bh = q8_scale_byte(group_max<LANES>(mh));
    const float il = q8_inv_scale(bl), ih = q8_inv_scale(bh);
    int8_t* cp = a.codes + ((int64_t)row * a.H + h) * 64 + l * V;
    Codes<V> wl, wh;
#pragma unroll
    for (int e = 0; e < V / 4; ++e) {
      wl.w[e] = bl == 255u ? 0u : q8_codes4(lo[4 * e], lo[4 * e + 1], lo[4 * e + 2], lo[4 * e + 3], il);
      wh.w[e] = bh == 255u ? 0u : q8_codes4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3], ih);
    }
    *reinterpret_cast<Codes<V>*>(cp) = wl;
    *reinterpret_cast<Codes<V>*>(cp + 32) = wh;
    if (l == 0) *reinterpret_cast<uint16_t*>(a.scales + ((int64_t)row * a.H + h) * 2) = (uint16_t)(bl | (bh << 8));
  }
  if constexpr (NORM) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) sq = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], sq));
    const float r = inv_rms<T, LANES>(sq, a.eps);
    const float* g = (h < a.Hq ? a.gq : a.gk) + l * V;
    float gl[V], gh[V];
    ld_f32<V>(g, gl);
    ld_f32<V>(g + 32, gh);
#pragma unroll
    for (int e = 0; e < V; ++e) { lo[e] = lo[e] * r * gl[e]; hi[e] = hi[e] * r * gh[e]; }
  }
  if constexpr (ROPE) {
    const int64_t t = (int64_t)(row % a.period) * 32 + l * V;
    float c[V], s[V];
    ld_f32<V>(a.cos + t, c);
    ld_f32<V>(a.sin + t, s);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float p = lo[e], q = hi[e];
      lo[e] = fmaf(p, c[e], -(q * s[e]));
      hi[e] = fmaf(q, c[e], p * s[e]);
    }
  }
  T* yp = reinterpret_cast<T*>(a.y) + (int64_t)row * a.ldy + h * 64 + l * V;
  st_vals<T, V>(yp, lo);
  st_vals<T, V>(yp + 32, hi);
}

// Backward.  A block takes heads of one kind (so that a lane's 2 V gain gradients stay in registers over all its heads) and leaves
// one row of 64 partial sums; qk_gain_kernel joins them in the order of the blocks: the result does not depend on timing.
template <typename T, bool NORM, bool ROPE, bool PACK>
__global__ __launch_bounds__(256) void qk_bwd_kernel(const QkArgs a) {
  constexpr int V = PACK ? 16 / sizeof(T) : 4, LANES = 32 / V, PER = 256 / LANES;
  const int l = threadIdx.x & (LANES - 1);
  const bool key = (int)blockIdx.x >= a.bq;
  const uint32_t nh = (uint32_t)(key ? a.H - a.Hq : a.Hq), h0 = (uint32_t)(key ? a.Hq : 0);
  const uint32_t b = key ? blockIdx.x - a.bq : blockIdx.x, nb = key ? gridDim.x - a.bq : a.bq;
  const uint32_t items = a.rows * nh;
  float gl[V], gh[V], dgl[V], dgh[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { gl[e] = gh[e] = 1.f; dgl[e] = dgh[e] = 0.f; }
  if constexpr (NORM) {
    const float* g = (key ? a.gk : a.gq) + l * V;
    ld_f32<V>(g, gl);
    ld_f32<V>(g + 32, gh);
  }
  for (uint32_t it = b * PER + threadIdx.x / LANES; it < items; it += nb * PER) {
    const uint32_t row = it / nh;
    const uint32_t h = h0 + (it - row * nh);
    const T* dp = reinterpret_cast<const T*>(a.dy) + (int64_t)row * a.lddy + h * 64 + l * V;
    float lo[V], hi[V], xl[V], xh[V];
    const Vals<T, V> d0 = ld_vals<V>(dp), d1 = ld_vals<V>(dp + 32);
    if constexpr (NORM && !PACK) {
      const T* xp = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx + h * 64 + l * V;
      unpack(ld_vals<V>(xp), xl);
      unpack(ld_vals<V>(xp + 32), xh);
    } else if constexpr (NORM) {
      const int64_t hd = (int64_t)row * a.H + h;
      const int8_t* cp = a.codes + hd * 64 + l * V;
      const uint32_t by = *reinterpret_cast<const uint16_t*>(a.scales + hd * 2);
      const float sl = q8_scale(by & 255u), sh = q8_scale(by >> 8);
      const Codes<V> wl = *reinterpret_cast<const Codes<V>*>(cp), wh = *reinterpret_cast<const Codes<V>*>(cp + 32);
#pragma unroll
      for (int e = 0; e < V; ++e) { xl[e] = q8_code(wl.w[e / 4], e & 3) * sl; xh[e] = q8_code(wh.w[e / 4], e & 3) * sh; }
    }
    unpack(d0, lo);
    unpack(d1, hi);
    if constexpr (ROPE) {
      const int64_t t = (int64_t)(row % a.period) * 32 + l * V;
      float c[V], s[V];
      ld_f32<V>(a.cos + t, c);
      ld_f32<V>(a.sin + t, s);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float p = lo[e], q = hi[e];
        lo[e] = fmaf(p, c[e], q * s[e]);
        hi[e] = fmaf(q, c[e], -(p * s[e]));
      }
    }
    if constexpr (NORM) {
      float sq = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) sq = fmaf(xl[e], xl[e], fmaf(xh[e], xh[e], sq));
      const float r = inv_rms<T, LANES>(sq, a.eps);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xl[e] *= r; xh[e] *= r;                            // u
        dgl[e] = fmaf(lo[e], xl[e], dgl[e]);
        dgh[e] = fmaf(hi[e], xh[e], dgh[e]);
        lo[e] *= gl[e]; hi[e] *= gh[e];                    // dz g
        dot = fmaf(lo[e], xl[e], fmaf(hi[e], xh[e], dot));
      }
      const float m = group_sum<LANES>(dot) * (1.f / 64.f);
#pragma unroll
      for (int e = 0; e < V; ++e) { lo[e] = r * fmaf(-xl[e], m, lo[e]); hi[e] = r * fmaf(-xh[e], m, hi[e]); }
    }
    T* yp = reinterpret_cast<T*>(a.y) + (int64_t)row * a.ldy + h * 64 + l * V;
    st_vals<T, V>(yp, lo);
    st_vals<T, V>(yp + 32, hi);
  }
  if constexpr (NORM) {
    __shared__ float sum[4][64];
#pragma unroll
    for (int e = 0; e < V; ++e)
#pragma unroll
      for (int o = LANES; o < 64; o <<= 1) {
        dgl[e] += __shfl_xor(dgl[e], o, 64);
        dgh[e] += __shfl_xor(dgh[e], o, 64);
      }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < LANES) {
#pragma unroll
      for (int e = 0; e < V; ++e) { sum[wave][l * V + e] = dgl[e]; sum[wave][32 + l * V + e] = dgh[e]; }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      const int c = threadIdx.x;
      a.part[(int64_t)blockIdx.x * 64 + c] = (sum[0][c] + sum[1][c]) + (sum[2][c] + sum[3][c]);
    }
  }
}

// gain gradients from the blocks' partial sums: block = (kind, four of the 64 channels), its threads over the partial sums
__global__ __launch_bounds__(256) void qk_gain_kernel(const float* __restrict__ part, int bq, int blocks, float* __restrict__ dgq,
                                                      float* __restrict__ dgk, int accumulate) {
  __shared__ f32x4 sum[4];
  const bool key = blockIdx.x >= 16;
  const int c = (blockIdx.x & 15) * 4, end = key ? blocks : bq;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int b = (key ? bq : 0) + threadIdx.x; b < end; b += 256) s += *reinterpret_cast<const f32x4*>(part + (int64_t)b * 64 + c);
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = wave_sum(s[e]);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x < 4) {
    const int e = threadIdx.x;
    const float v = (sum[0][e] + sum[1][e]) + (sum[2][e] + sum[3][e]);
    float* o = (key ? dgk : dgq) + c + e;
    *o = accumulate ? *o + v : v;
  }
}

// heads that a block of the backward takes at a time, and blocks for the heads of one kind: `most` in all at most, in proportion, each with
// at least one full turn of its lanes.  (Measured in bf16, 16,400 rows x 24 heads from the checkpoint: 1,024 blocks 25.8 us, 768 26.3, 2,048
// 26.8, 4,096 30.2; from x 768 27.8 us, 1,024 28.4, 512 28.2, 2,048 28.7: the blocks end with a reduction and leave 256 bytes each to be joined.)
int bwd_heads(bool packed, int dtype) { return packed && dtype == S4F_BF16 ? 64 : 32; }
int bwd_most(bool packed) { return packed ? 1024 : 768; }
int bwd_blocks(int64_t rows, int64_t heads, int64_t all, int per, int most) {
  const int64_t b = (rows * heads + per - 1) / per, cap = std::max<int64_t>(1, most * heads / all);
  return (int)std::min(b, cap);
}

int check_qk(const char* who, int64_t rows, int Hq, int Hk, int dtype, const float* gq, const float* gk, const float* cos,
             const float* sin, int64_t period, float eps) {
  S4F_CHECK(dtype == S4F_F32 || dtype == S4F_BF16, "%s: bad dtype %d", who, dtype);
  S4F_CHECK(rows > 0 && Hq > 0 && Hk > 0, "%s: rows=%lld, Hq=%d, Hk=%d must be positive", who, (long long)rows, Hq, Hk);
  S4F_CHECK(rows < (1LL << 31) && rows * ((int64_t)Hq + Hk) < (1LL << 31) - (1 << 22), "%s: rows x heads must stay below 2^31 - 2^22", who);
  S4F_CHECK((gq != nullptr) == (gk != nullptr) && (cos != nullptr) == (sin != nullptr), "%s: gains and tables come in pairs", who);
  S4F_CHECK(gq || cos, "%s: neither a norm (gains) nor a rotation (tables) asked for", who);
  // (the hardware's reciprocal root takes a denormal argument for zero: a row of zeros would become 0 x infinity)
  S4F_CHECK(!gq || (eps >= FLT_MIN && eps <= 1e30f), "%s: eps must be finite and at least the least normal fp32 number", who);
  S4F_CHECK(!cos || (period > 0 && period <= rows && rows % period == 0), "%s: the tables' %lld positions must divide the %lld rows", who,
            (long long)period, (long long)rows);
  for (const void* p : {(const void*)gq, (const void*)gk, (const void*)cos, (const void*)sin})
    S4F_CHECK((uintptr_t)p % 16 == 0, "%s: gains and tables must be 16-byte aligned", who);
  return 0;
}
// a piece of `written` has a byte in common with a gain or a table
bool meet_params(const float* gq, const float* gk, const float* cos, const float* sin, int64_t period, std::initializer_list<Piece> written) {
  const int64_t tab = cos ? period * 32 * 4 : 0;
  for (const Piece& w : written)
    if (meet(w, {piece(gq, 256), piece(gk, 256), piece(cos, tab), piece(sin, tab)})) return true;
  return false;
}
int check_rows(const char* who, const char* what, const void* p, int64_t ld, int dtype) {
  S4F_CHECK(p, "%s: %s is null", who, what);
  S4F_CHECK((uintptr_t)p % 16 == 0 && ld >= 0 && ld % (dtype == S4F_BF16 ? 8 : 4) == 0, "%s: rows of %s must start on 16-byte boundaries", who, what);
  return 0;
}

template <typename T> void launch_fwd(const QkArgs& a, hipStream_t st) {
  constexpr int PER = 256 / (32 / (16 / (int)sizeof(T)));
  const dim3 grid((unsigned)(((int64_t)a.rows * a.H + PER - 1) / PER));
  const bool n = a.gq, r = a.cos, p = a.codes;
#define GO(N, R, P) hipLaunchKernelGGL((qk_fwd_kernel<T, N, R, P>), grid, dim3(256), 0, st, a)
  if (n && r) { if (p) GO(true, true, true); else GO(true, true, false); }
  else if (n) { if (p) GO(true, false, true); else GO(true, false, false); }
  else GO(false, true, false);
#undef GO
}
template <typename T> void launch_bwd(const QkArgs& a, int blocks, hipStream_t st) {
  const bool n = a.gq, r = a.cos, p = a.codes;
#define GO(N, R, P) hipLaunchKernelGGL((qk_bwd_kernel<T, N, R, P>), dim3(blocks), dim3(256), 0, st, a)
  if (n && r) { if (p) GO(true, true, true); else GO(true, true, false); }
  else if (n) { if (p) GO(true, false, true); else GO(true, false, false); }
  else GO(false, true, false);
#undef GO
}

}  // namespace

S4F_API int s4f_qk_norm_rope_fwd(const void* x, int64_t ldx, void* y, int64_t ldy, const float* gq, const float* gk, const float* cos,
                                 const float* sin, int64_t period, float eps, int8_t* codes, uint8_t* scales, int64_t rows, int Hq,
                                 int Hk, int dtype, s4f_stream stream) {
  const char* who = "s4f_qk_norm_rope_fwd";
  if (int rc = check_qk(who, rows, Hq, Hk, dtype, gq, gk, cos, sin, period, eps)) return rc;
  if (int rc = check_rows(who, "x", x, ldx, dtype)) return rc;
  if (int rc = check_rows(who, "y", y, ldy, dtype)) return rc;
  S4F_CHECK(rows == 1 || ldy >= (int64_t)(Hq + Hk) * 64, "%s: rows of y overlap", who);
  // (a launch has at most 2^32 - 1 threads; a head takes 4 or 8 of them.  128 GiB of T)
  S4F_CHECK(rows * (Hq + Hk) <= (dtype == S4F_BF16 ? 1LL << 30 : 1LL << 29) - 64, "%s: rows x heads too large for one launch", who);
  S4F_CHECK((codes != nullptr) == (scales != nullptr) && (!codes || gq), "%s: a checkpoint needs codes, scales and the norm", who);
  S4F_CHECK((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 2 == 0, "%s: codes / scales alignment (16 / 2 bytes)", who);
  const int64_t C = (int64_t)(Hq + Hk) * 64;
  const int es = dtype == S4F_BF16 ? 2 : 4;
  const Piece px = piece(x, rows, ldx, C, es), py = piece(y, rows, ldy, C, es), pc = piece(codes, rows * C), ps = piece(scales, rows * C / 32);
  S4F_CHECK(same_or_apart(x, ldx, y, ldy, rows, C, es), "%s: x and y overlap", who);
  S4F_CHECK(!meet(pc, {px, py, ps}) && !meet(ps, {px, py}), "%s: the checkpoint overlaps x or y", who);
  S4F_CHECK(!meet_params(gq, gk, cos, sin, period, {py, pc, ps}), "%s: y or the checkpoint overlaps the gains or the tables", who);
  QkArgs a{};
  a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.gq = gq; a.gk = gk; a.cos = cos; a.sin = sin; a.codes = codes; a.scales = scales;
  a.eps = eps; a.rows = (uint32_t)rows; a.period = (uint32_t)(cos ? period : 1); a.Hq = Hq; a.H = Hq + Hk;
  if (dtype == S4F_BF16) launch_fwd<bf16_t>(a, (hipStream_t)stream); else launch_fwd<float>(a, (hipStream_t)stream);
  S4F_LAUNCH_CHECK();
  return 0;
}

int64_t s4f_qk_ws_bytes(int64_t rows, int Hq, int Hk) {
  if (rows <= 0 || rows >= (1LL << 31) || Hq <= 0 || Hk <= 0) return -1;
  return ((int64_t)bwd_blocks(rows, Hq, (int64_t)Hq + Hk, 32, 1024) + bwd_blocks(rows, Hk, (int64_t)Hq + Hk, 32, 1024)) * 64 * 4;
}

S4F_API int s4f_qk_norm_rope_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const int8_t* codes, const uint8_t* scales,
                                 void* dx, int64_t lddx, const float* gq, const float* gk, const float* cos, const float* sin,
                                 int64_t period, float eps, float* dgq, float* dgk, int accumulate, void* ws, int64_t ws_bytes,
                                 int64_t rows, int Hq, int Hk, int dtype, s4f_stream stream) {
  const char* who = "s4f_qk_norm_rope_bwd";
  if (int rc = check_qk(who, rows, Hq, Hk, dtype, gq, gk, cos, sin, period, eps)) return rc;
  if (int rc = check_rows(who, "dy", dy, lddy, dtype)) return rc;
  if (int rc = check_rows(who, "dx", dx, lddx, dtype)) return rc;
  S4F_CHECK(rows == 1 || lddx >= (int64_t)(Hq + Hk) * 64, "%s: rows of dx overlap", who);
  const int64_t C = (int64_t)(Hq + Hk) * 64;
  const int es = dtype == S4F_BF16 ? 2 : 4;
  const Piece pd = piece(dx, rows, lddx, C, es), pw = piece(gq ? ws : nullptr, ws_bytes), pq = piece(gq ? dgq : nullptr, 256),
              pk = piece(gq ? dgk : nullptr, 256);
  if (gq) {
    S4F_CHECK((codes != nullptr) == (scales != nullptr) && (codes != nullptr) != (x != nullptr), "%s: the norm's backward needs x or its checkpoint, not both", who);
    if (!codes)
      if (int rc = check_rows(who, "x", x, ldx, dtype)) return rc;
    S4F_CHECK((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 2 == 0, "%s: codes / scales alignment (16 / 2 bytes)", who);
    S4F_CHECK(dgq && dgk && ws && (uintptr_t)ws % 16 == 0, "%s: gain gradients and a 16-byte aligned workspace needed", who);
    S4F_CHECK(ws_bytes >= s4f_qk_ws_bytes(rows, Hq, Hk), "%s: workspace too small (%lld < %lld)", who, (long long)ws_bytes,
              (long long)s4f_qk_ws_bytes(rows, Hq, Hk));
    const Piece pc = piece(codes, rows * C), ps = piece(scales, rows * C / 32), py = piece(dy, rows, lddy, C, es), px = piece(x, rows, ldx, C, es);
    S4F_CHECK(!meet(pd, {pc, ps, pw, pq, pk}) && !meet(pw, {py, px, pc, ps, pq, pk}) && !meet(pq, {pk, py, px, pc, ps}) && !meet(pk, {py, px, pc, ps}),
              "%s: dx, the gain gradients or the workspace overlap each other or an input", who);
    S4F_CHECK(codes || same_or_apart(x, ldx, dx, lddx, rows, C, es), "%s: x and dx overlap", who);
  }
  S4F_CHECK(same_or_apart(dy, lddy, dx, lddx, rows, C, es), "%s: dy and dx overlap", who);
  S4F_CHECK(!meet_params(gq, gk, cos, sin, period, {pd, pw, pq, pk}), "%s: dx, the gain gradients or the workspace overlap the gains or the tables", who);
  QkArgs a{};
  a.dy = dy; a.lddy = lddy; a.x = x; a.ldx = ldx; a.y = dx; a.ldy = lddx; a.gq = gq; a.gk = gk; a.cos = cos; a.sin = sin;
  a.codes = gq ? const_cast<int8_t*>(codes) : nullptr; a.scales = const_cast<uint8_t*>(scales); a.part = (float*)ws; a.eps = eps;
  a.rows = (uint32_t)rows; a.period = (uint32_t)(cos ? period : 1); a.Hq = Hq; a.H = Hq + Hk;
  const int per = bwd_heads(a.codes, dtype), most = bwd_most(a.codes);
  a.bq = bwd_blocks(rows, Hq, Hq + Hk, per, most);
  const int blocks = a.bq + bwd_blocks(rows, Hk, Hq + Hk, per, most);
  if (dtype == S4F_BF16) launch_bwd<bf16_t>(a, blocks, (hipStream_t)stream); else launch_bwd<float>(a, blocks, (hipStream_t)stream);
  S4F_LAUNCH_CHECK();
  if (gq) {
    hipLaunchKernelGGL(qk_gain_kernel, dim3(32), dim3(256), 0, (hipStream_t)stream, (const float*)ws, a.bq, blocks, dgq, dgk, accumulate);
    S4F_LAUNCH_CHECK();
  }
  return 0;
}
