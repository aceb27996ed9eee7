// Weight gradients of linear layers whose inputs are 8-bit activation checkpoints (actq8.h): s4f_wgrad_packed.
//   dW[m][n] (+)= sum_r dY[r][m] code[r][n] s[r][n / 32]
// code * s is exact in bf16, so the products of a bf16 dY are the products of the restored activations, summed in fp32 by the matrix
// units.  Up to four problems (the layers of one encoder block) share a grid.
//
// The rows are cut into ranges so that the grid fills the chip; a range's sums go to a slab of the workspace with plain stores and
// wgrad_join_kernel adds the slabs in the order of the ranges: the result does not depend on timing.
#include "actq8.h"
#include "../../include/s4f.h"
#include <algorithm>

static_assert(sizeof(s4f_wgrad_packed_desc) == 56, "mirrored by _lib.WgradPackedDesc");

namespace {

constexpr int MAXP = 4;

struct Problem {
  const void* dy; int64_t lddy;
  const int8_t* codes; const uint8_t* scales;
  float* out;                            // [M][N]
  float* slab;                           // [splits][M][N], splits > 1
  int64_t rows;
  int M, N, tiles_n, tiles, splits, steps, steps_per_split;
  int work_end;                          // running sum of tiles x splits
};
struct Args { Problem p[MAXP]; int count, accumulate; };

// ------------------------------------------------------------------------------------------------- 128 x 128 tile, any type
constexpr int BT = 128, BKR = 32;
template <typename T> constexpr int lds_stride() { return BT * (int)sizeof(T) + 16; }

template <typename T>
__global__ __launch_bounds__(256) void wgrad_kernel(const Args args) {
  constexpr int V = 16 / sizeof(T), NA = BKR * (BT / V) / 256, LD = lds_stride<T>();
  __shared__ __attribute__((aligned(16))) char smem[2 * BKR * LD];
  char* const la = smem;
  char* const lb = smem + BKR * LD;

  int which = 0;
  for (int i = 0; i < MAXP - 1; ++i) which += i < args.count - 1 && (int)blockIdx.x >= args.p[i].work_end ? 1 : 0;
  const Problem& P = args.p[which];
  const int local = (int)blockIdx.x - (which ? args.p[which - 1].work_end : 0);
  const int z = local / P.tiles, tile = local - z * P.tiles;
  const int m0 = tile / P.tiles_n * BT, n0 = tile % P.tiles_n * BT;
  const int k_beg = z * P.steps_per_split, k_end = min(k_beg + P.steps_per_split, P.steps);

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, g = l >> 4, li = l & 15;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const T* dy = reinterpret_cast<const T*>(P.dy);
  const int N = P.N, M = P.M;

  chunk16 ra[NA], rb;
  uint32_t rs;
  auto load = [&](int k) {
    const int64_t r0 = (int64_t)k * BKR;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int c = tid + i * 256, row = c / (BT / V), col = (c % (BT / V)) * V;
      const bool ok = r0 + row < P.rows && m0 + col < M;     // (M is a multiple of 8: a chunk is inside or outside)
      ra[i] = ok ? ld_global16(dy + (r0 + row) * P.lddy + m0 + col) : zero16();
    }
    const int row = tid >> 3, col = (tid & 7) * 16;
    const bool ok = r0 + row < P.rows && n0 + col < N;
    rb = ok ? ld_global16(P.codes + (r0 + row) * N + n0 + col) : zero16();
    rs = ok ? P.scales[(r0 + row) * (N / ACTQ8_GROUP) + (n0 + col) / ACTQ8_GROUP] : 0u;
  };
  auto store = [&]() {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int c = tid + i * 256, row = c / (BT / V), col = (c % (BT / V)) * V;
      *reinterpret_cast<chunk16*>(la + row * LD + col * (int)sizeof(T)) = ra[i];
    }
    const float s = q8_scale(rs);
    char* o = lb + (tid >> 3) * LD + (tid & 7) * 16 * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += V) {
      chunk16 c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (V == 8) c.w[e] = pack_exact_bf16(q8_code(rb.w[(i + 2 * e) / 4], (2 * e) & 3) * s, q8_code(rb.w[(i + 2 * e) / 4], (2 * e + 1) & 3) * s);
        else c.w[e] = __float_as_uint(q8_code(rb.w[i / 4], e) * s);
      }
      *reinterpret_cast<chunk16*>(o + i * (int)sizeof(T)) = c;
    }
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (k_beg < k_end) load(k_beg);
  for (int k = k_beg; k < k_end; ++k) {
    __syncthreads();
    store();
    __syncthreads();
    if (k + 1 < k_end) load(k + 1);
    Frag<T> b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) lds_read_tr(b[j], lb, LD, 0, wn + j * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Frag<T> a;
      lds_read_tr(a, la, LD, 0, wm + i * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mma16(a, b[j], acc[i][j]);
    }
  }

  const bool add = P.splits == 1 && args.accumulate;
  float* o = P.splits == 1 ? P.out : P.slab + (int64_t)z * M * N;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + wn + j * 16 + li;
      if (n >= N) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + wm + i * 16 + 4 * g + r;
        if (m >= M) continue;
        float* q = o + (int64_t)m * N + n;
        *q = add ? *q + acc[i][j][r] : acc[i][j][r];
      }
    }
}

// out (+)= the slabs in the order of the row ranges
__global__ __launch_bounds__(256) void wgrad_join_kernel(const Args args) {
  for (int i = 0; i < args.count; ++i) {
    const Problem& P = args.p[i];
    if (P.splits == 1) continue;
    const int64_t n4 = (int64_t)P.M * P.N / 4;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n4; e += (int64_t)gridDim.x * 256) {
      f32x4 s = args.accumulate ? reinterpret_cast<const f32x4*>(P.out)[e] : f32x4{0.f, 0.f, 0.f, 0.f};
      for (int z = 0; z < P.splits; ++z) s += reinterpret_cast<const f32x4*>(P.slab)[z * n4 + e];
      reinterpret_cast<f32x4*>(P.out)[e] = s;
    }
  }
}

// tiles and row ranges of the problems; returns the bytes of slabs, or -1
int64_t plan(Args& a, int dtype) {
  int64_t tiles = 0;
  for (int i = 0; i < a.count; ++i) {
    Problem& p = a.p[i];
    if (p.M <= 0 || p.N <= 0 || p.rows <= 0 || p.M % 8 || p.N % ACTQ8_GROUP || p.rows > (1LL << 31) || (int64_t)p.M * p.N > (1LL << 31)) return -1;
    p.tiles_n = ceil_div(p.N, BT);
    p.tiles = ceil_div(p.M, BT) * p.tiles_n;
    tiles += p.tiles;
  }
  int64_t bytes = 0, work = 0;
  for (int i = 0; i < a.count; ++i) {
    Problem& p = a.p[i];
    p.steps = ceil_div(p.rows, BKR);
    int64_t s = (512 + tiles / 2) / tiles;
    if (s > p.steps / 8) s = p.steps / 8;
    if (s < 1) s = 1;
    p.steps_per_split = ceil_div(p.steps, s);
    p.splits = ceil_div(p.steps, p.steps_per_split);
    work += (int64_t)p.tiles * p.splits;
    p.work_end = (int)work;
    if (p.splits > 1) {
      p.slab = reinterpret_cast<float*>(bytes);            // offset, resolved against the workspace by the caller
      bytes += (int64_t)p.splits * p.M * p.N * 4;
    }
  }
  return work < (1LL << 31) ? bytes : -1;
}

}  // namespace

// dims: {dtype, then M, N, rows of each problem}
int64_t s4f_wgrad_packed_ws(const int64_t* dims, int ndims) {
  if (ndims < 4 || (ndims - 1) % 3 || (ndims - 1) / 3 > MAXP) return -1;
  Args a{};
  a.count = (ndims - 1) / 3;
  for (int i = 0; i < a.count; ++i) {
    const int64_t* d = dims + 1 + 3 * i;
    if (d[0] > INT32_MAX || d[1] > INT32_MAX) return -1;
    a.p[i].M = (int)d[0]; a.p[i].N = (int)d[1]; a.p[i].rows = d[2];
  }
  return plan(a, (int)dims[0]);
}

S4F_API int s4f_wgrad_packed(const s4f_wgrad_packed_desc* descs, int count, int dtype, int accumulate, void* ws, int64_t ws_bytes,
                             s4f_stream stream) {
  const char* who = "s4f_wgrad_packed";
  S4F_CHECK(dtype == S4F_F32 || dtype == S4F_BF16, "%s: bad dtype %d", who, dtype);
  S4F_CHECK(descs && count >= 1 && count <= MAXP, "%s: 1..%d problems", who, MAXP);
  Args a{};
  a.count = count;
  a.accumulate = accumulate;
  for (int i = 0; i < count; ++i) {
    const s4f_wgrad_packed_desc& d = descs[i];
    S4F_CHECK(d.dy && d.codes && d.scales && d.out, "%s: null pointer in problem %d", who, i);
    S4F_CHECK((uintptr_t)d.dy % 16 == 0 && (uintptr_t)d.codes % 16 == 0 && (uintptr_t)d.out % 16 == 0 && d.lddy >= 0 &&
                  d.lddy % (dtype == S4F_BF16 ? 8 : 4) == 0, "%s: rows of dy, codes and out must start on 16-byte boundaries (problem %d)", who, i);
    S4F_CHECK(d.M > 0 && d.N > 0 && d.rows > 0 && d.M % 8 == 0 && d.N % ACTQ8_GROUP == 0,
              "%s: M=%d must be a multiple of 8, N=%d of 32, rows=%lld positive", who, d.M, d.N, (long long)d.rows);
    Problem& p = a.p[i];
    p.dy = d.dy; p.lddy = d.lddy; p.codes = d.codes; p.scales = d.scales; p.out = d.out; p.M = d.M; p.N = d.N; p.rows = d.rows;
  }
  const int64_t need = plan(a, dtype);
  S4F_CHECK(need >= 0, "%s: sizes too large for one launch", who);
  S4F_CHECK(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need), "%s: workspace missing, misaligned or too small (%lld < %lld)",
            who, (long long)ws_bytes, (long long)need);
  bool join = false;
  int64_t n4 = 0;
  for (int i = 0; i < count; ++i)
    if (a.p[i].splits > 1) {
      a.p[i].slab = reinterpret_cast<float*>((char*)ws + (int64_t)reinterpret_cast<uintptr_t>(a.p[i].slab));
      join = true;
      n4 = std::max<int64_t>(n4, (int64_t)a.p[i].M * a.p[i].N / 4);
    }
  const dim3 grid(a.p[count - 1].work_end);
  if (dtype == S4F_BF16) hipLaunchKernelGGL(wgrad_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(wgrad_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
  S4F_LAUNCH_CHECK();
  if (join) {
    hipLaunchKernelGGL(wgrad_join_kernel, dim3((unsigned)std::min<int64_t>((n4 + 255) / 256, 2048)), dim3(256), 0, (hipStream_t)stream, a);
    S4F_LAUNCH_CHECK();
  }
  return 0;
}
