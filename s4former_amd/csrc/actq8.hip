// Activation checkpoints in 8 bits (actq8.h has the format): s4f_act_pack, s4f_act_unpack.
//
// Both are one pass bound by HBM: 16 bytes of T per lane and access (8 bf16 / 4 fp32), a group of 32 spread over 4 / 8 lanes, so
// that a wave reads and writes whole lines and the group's maximum takes two or three lane exchanges without LDS.
// Measured at 8,200 x 4,096, calls one behind the other on the same tensors (in the last-level cache) / on fresh ones: bf16 pack 16.1 /
// 20.2 us, unpack 15.3 / 21.5 us (6.3 and 6.7 / 5.0 and 4.7 TB/s; a large copy 4.8 - 5.0), fp32 pack 24.4 / 31.0 us, unpack 25.5 / 33.3 us.
#include "actq8.h"
#include "../../include/s4f.h"

namespace {

constexpr int UNR = 4;                                     // chunks per thread, their loads in flight together

template <typename T> __device__ __forceinline__ void unpack16(const chunk16& c, float (&v)[16 / sizeof(T)]);
template <> __device__ __forceinline__ void unpack16<float>(const chunk16& c, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(c.w[i]);
}
template <> __device__ __forceinline__ void unpack16<bf16_t>(const chunk16& c, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(c.w[i] << 16);
    v[2 * i + 1] = __uint_as_float(c.w[i] & 0xffff0000u);
  }
}

// chunk i (16 bytes of T) of the matrix -> element offset in a [rows, ld] buffer; STRIDED: ld != C
template <bool STRIDED, int V> __device__ __forceinline__ int64_t elem_of(int64_t i, uint32_t cpr, int64_t ld) {
  if constexpr (!STRIDED) return i * V;
  const uint32_t row = (uint32_t)i / cpr, col = (uint32_t)i - row * cpr;
  return (int64_t)row * ld + (int64_t)col * V;
}

template <typename T, bool STRIDED>
__global__ __launch_bounds__(256) void act_pack_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, int64_t chunks, uint32_t cpr) {
  constexpr int V = 16 / sizeof(T), LANES = 32 / V;
  const int64_t i0 = (int64_t)blockIdx.x * (256 * UNR) + threadIdx.x;
  chunk16 c[UNR];
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const int64_t i = i0 + u * 256;
    c[u] = i < chunks ? ld_global16(x + elem_of<STRIDED, V>(i, cpr, ldx)) : zero16();
  }
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const int64_t i = i0 + u * 256;
    float v[V];
    unpack16<T>(c[u], v);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) m = max(m, mag_bits(v[e]));
    const uint32_t byte = q8_scale_byte(group_max<LANES>(m));
    const float inv = q8_inv_scale(byte);
    uint32_t w[V / 4];
#pragma unroll
    for (int e = 0; e < V / 4; ++e) {
      w[e] = q8_codes4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3], inv);
      if (byte == 255u) w[e] = 0;
    }
    if (i < chunks) {
      if constexpr (V == 8) *reinterpret_cast<uint2*>(codes + i * V) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(codes + i * V) = w[0];
      if ((threadIdx.x & (LANES - 1)) == 0) scales[i / LANES] = (uint8_t)byte;
    }
  }
}

template <typename T, bool STRIDED>
__global__ __launch_bounds__(256) void act_unpack_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                         T* __restrict__ y, int64_t ldy, int64_t chunks, uint32_t cpr) {
  constexpr int V = 16 / sizeof(T), LANES = 32 / V;
  const int64_t i0 = (int64_t)blockIdx.x * (256 * UNR) + threadIdx.x;
  uint32_t w[UNR][V / 4];
  uint32_t b[UNR];
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const int64_t i = i0 + u * 256;
    const bool ok = i < chunks;
    if constexpr (V == 8) {
      const uint2 q = ok ? *reinterpret_cast<const uint2*>(codes + i * V) : make_uint2(0, 0);
      w[u][0] = q.x; w[u][1] = q.y;
    } else {
      w[u][0] = ok ? *reinterpret_cast<const uint32_t*>(codes + i * V) : 0;
    }
    b[u] = ok ? scales[i / LANES] : 0;
  }
#pragma unroll
  for (int u = 0; u < UNR; ++u) {
    const int64_t i = i0 + u * 256;
    if (i >= chunks) continue;
    const float s = q8_scale(b[u]);
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = q8_code(w[u][e / 4], e & 3) * s;
    chunk16 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.w[e] = V == 8 ? pack_exact_bf16(v[(2 * e) % V], v[(2 * e + 1) % V]) : __float_as_uint(v[e]);
    *reinterpret_cast<chunk16*>(y + elem_of<STRIDED, V>(i, cpr, ldy)) = o;
  }
}

// what both entry points check: whole groups, 16-byte rows, an index that fits the strided form's 32-bit division
int check_extent(const char* who, const void* t, int64_t ld, const void* codes, const void* scales, int64_t rows, int64_t C, int dtype) {
  S4F_CHECK(dtype == S4F_F32 || dtype == S4F_BF16, "%s: bad dtype %d", who, dtype);
  S4F_CHECK(t && codes && scales, "%s: null pointer", who);
  S4F_CHECK(rows > 0 && C > 0 && C % ACTQ8_GROUP == 0, "%s: C=%lld must be a positive multiple of 32, rows=%lld positive", who, (long long)C, (long long)rows);
  const int ts = dtype == S4F_BF16 ? 2 : 4;
  S4F_CHECK(ld >= 0 && (ld * ts) % 16 == 0 && (uintptr_t)t % 16 == 0 && (uintptr_t)codes % 16 == 0, "%s: rows and codes must start on 16-byte boundaries", who);
  const int64_t cpr = C / (16 / ts);
  S4F_CHECK(rows <= (int64_t)0xffffff * 256 * UNR / cpr, "%s: rows=%lld too large for one launch", who, (long long)rows);
  S4F_CHECK(ld == C || rows <= (int64_t)0xffffffffu / cpr, "%s: rows=%lld too large for a strided view", who, (long long)rows);
  const Piece c = piece(codes, rows * C), s = piece(scales, rows * (C / ACTQ8_GROUP));
  S4F_CHECK(!meet(piece(t, rows, ld, C, ts), {c, s}) && !meet(c, s), "%s: the activation, its codes and its scales overlap", who);
  return 0;
}

}  // namespace

S4F_API int s4f_act_pack(const void* x, int64_t ldx, int8_t* codes, uint8_t* scales, int64_t rows, int C, int dtype, s4f_stream stream) {
  if (int rc = check_extent("s4f_act_pack", x, ldx, codes, scales, rows, C, dtype)) return rc;
  const uint32_t cpr = (uint32_t)(C / (dtype == S4F_BF16 ? 8 : 4));
  const int64_t chunks = rows * cpr;
  const dim3 grid((unsigned)((chunks + 256 * UNR - 1) / (256 * UNR)));
#define PACK(T, S) hipLaunchKernelGGL((act_pack_kernel<T, S>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)x, ldx, codes, scales, chunks, cpr)
  if (dtype == S4F_BF16) { if (ldx == C) PACK(bf16_t, false); else PACK(bf16_t, true); }
  else { if (ldx == C) PACK(float, false); else PACK(float, true); }
#undef PACK
  S4F_LAUNCH_CHECK();
  return 0;
}

S4F_API int s4f_act_unpack(const int8_t* codes, const uint8_t* scales, void* y, int64_t ldy, int64_t rows, int C, int dtype, s4f_stream stream) {
  if (int rc = check_extent("s4f_act_unpack", y, ldy, codes, scales, rows, C, dtype)) return rc;
  S4F_CHECK(ldy >= C || rows == 1, "s4f_act_unpack: rows of y overlap (ld %lld < C %d)", (long long)ldy, C);
  const uint32_t cpr = (uint32_t)(C / (dtype == S4F_BF16 ? 8 : 4));
  const int64_t chunks = rows * cpr;
  const dim3 grid((unsigned)((chunks + 256 * UNR - 1) / (256 * UNR)));
#define UNPACK(T, S) hipLaunchKernelGGL((act_unpack_kernel<T, S>), grid, dim3(256), 0, (hipStream_t)stream, codes, scales, (T*)y, ldy, chunks, cpr)
  if (dtype == S4F_BF16) { if (ldy == C) UNPACK(bf16_t, false); else UNPACK(bf16_t, true); }
  else { if (ldy == C) UNPACK(float, false); else UNPACK(float, true); }
#undef UNPACK
  S4F_LAUNCH_CHECK();
  return 0;
}
