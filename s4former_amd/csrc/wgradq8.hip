// Weight gradients of linear layers whose inputs are 8-bit activation checkpoints (actq8.h): s4f_wgrad_packed.
//   dW[m][n] (+)= sum_r dY[r][m] code[r][n] s[r][n / 32]
// code * s is exact in bf16, so the products of a bf16 dY are the products of the restored activations, summed in fp32 by the matrix
// units.  Up to four problems (the layers of one encoder block) share a grid.
//
// The rows are cut into ranges so that the grid fills the chip; a range's sums go to a slab of the workspace with plain stores and
// a second kernel adds the slabs in the order of the ranges: the result does not depend on timing.
#include "actq8.h"
#include "../../include/s4f.h"
#include <algorithm>

static_assert(sizeof(s4f_wgrad_packed_desc) == 56, "mirrored by _lib.WgradPackedDesc");

namespace {

constexpr int MAXP = 4;

// Offsets into the rows of a step are unsigned.  A column outside the matrix gets OUTSIDE, which stays beyond every resource (at most 2^30
// bytes: 64 rows of 2^24 or 128 of 2^23) whatever is added for a later row of the step (less than 2^30) or taken for the other half of a chunk
constexpr uint32_t OUTSIDE = 0x80000000u, MOST = 1u << 30;
// 16 codes come as two halves of eight; where `hb`, the upper one first: offset of the second
constexpr uint32_t second_half(uint32_t first, int hb) { return hb ? first - 8 : first + 8; }
static_assert(second_half(OUTSIDE, 0) >= MOST && second_half(OUTSIDE, 1) >= MOST && second_half(OUTSIDE, 0) + MOST > OUTSIDE,
              "a column outside reads as zero from both halves, in every row of a step");

struct Problem {
  const void* dy; int64_t lddy;
  const int8_t* codes; const uint8_t* scales;
  float* out;                            // [M][N]
  float* slab;                           // splits > 1: partial sums, [splits][M][N] (fp32) or [splits][tiles] in register order (bf16)
  int64_t rows;
  int M, N, tiles_n, tiles, splits, steps, steps_per_split;
  int work_end;                          // running sum of tiles x splits
};
struct Args { Problem p[MAXP]; int count, accumulate, variant; };

// Work is numbered (problem, row range, tile).  Consecutive blocks go to the eight XCDs in turn; a contiguous eighth of the numbers a
// XCD lets the tiles of a row range, which read the same rows of dY and X, meet in one L2.
__device__ __forceinline__ int work_of_block(int total) {
  const int xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
  return min(xcd, r8) * (q8 + 1) + max(xcd - r8, 0) * q8 + ((int)blockIdx.x >> 3);
}

// ------------------------------------------------------------------------------------------------- fp32
// 64 x 64 tile, four waves with one product of 32 x 32 x 2 each, 64 rows a step, two buffers, two tiles a CU.  The fp32 matrix rate (256
// operations a clock and CU: 2,048 clocks a step) bounds large problems; the small tile keeps ragged sizes from wasting it.  Counters say
// that a SIMD issues no other vector instruction beside an fp32 product: 2,760 clocks a step with one block on a CU, 2,480 for each of
// two.  Measured: 768 x 768 over 16,400 rows 164 us (118 TFLOP/s), 520 x 416 over 2,307 rows 19 us with the join.
//
// LDS image: [16 groups of four rows][64 columns], a column's four rows in 16 bytes: a thread turns the 4 x 4 block that it loaded in
// its registers, and one 16-byte read a lane feeds four products.  Bits 3 and 4 of a column move its lower two, so that the
// stores, whose lanes are four columns apart, touch different banks (no conflicts are counted).
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
// everyone's accesses of LDS are done (loads that go there among them), those of registers need not be
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
constexpr int BT = 64, BKR = 64;
__device__ __forceinline__ int f32_place(int col) { return col ^ (col >> 3 & 3); }

__global__ __launch_bounds__(256, 2) void wgrad_f32_kernel(const Args args) {
  __shared__ u32x4 la[2][BKR / 4 * BT];
  __shared__ f32x4 lb[2][BKR / 4 * BT];                   // 64 KiB in all
  const int w = work_of_block(args.p[args.count - 1].work_end);
  int which = 0;
  for (int i = 0; i < MAXP - 1; ++i) which += i < args.count - 1 && w >= args.p[i].work_end ? 1 : 0;
  const Problem& P = args.p[which];
  const int local = w - (which ? args.p[which - 1].work_end : 0);
  const int z = local / P.tiles, tile = local - z * P.tiles;
  const int m0 = tile / P.tiles_n * BT, n0 = tile % P.tiles_n * BT;
  const int k_beg = z * P.steps_per_split, k_end = min(k_beg + P.steps_per_split, P.steps);
  const int N = P.N, M = P.M, ns = N / ACTQ8_GROUP;

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int wm = (wave >> 1) * 32 + (l & 31), wn = (wave & 1) * 32 + (l & 31);
  // a thread's block: rows 4 rg .. + 3, columns c4 .. + 3 of dY and of the codes (M is a multiple of 8 and N of 32: inside or outside).  The
  // resources cover the rows of the step, so rows behind the range read as zero; columns outside get an offset beyond every resource
  const int rg = tid >> 4, c4 = (tid & 15) * 4;
  const int ld4 = (int)(P.lddy * 4);
  const uint32_t va = m0 + c4 < M ? 4 * rg * ld4 + (m0 + c4) * 4 : OUTSIDE;
  const uint32_t vb = n0 + c4 < N ? 4 * rg * N + n0 + c4 : OUTSIDE;
  const uint32_t vs = n0 + c4 < N ? 4 * rg * ns + (n0 + c4) / ACTQ8_GROUP : OUTSIDE;
  const int64_t r_beg = (int64_t)k_beg * BKR;
  int left = (int)(min(P.rows, (int64_t)k_end * BKR) - r_beg);
  char* pa = (char*)P.dy + r_beg * ld4;
  char* pb = (char*)P.codes + r_beg * N;
  char* ps = (char*)P.scales + r_beg * ns;
  __amdgpu_buffer_rsrc_t qa, qb, qs;
  auto next_rows = [&]() {                                 // the resources of the next step's rows (none left: empty ones)
    const int nr = __builtin_amdgcn_readfirstlane(max(min(left, BKR), 0));
    qa = __builtin_amdgcn_make_buffer_rsrc(pa, 0, nr * ld4, 0x00020000);
    qb = __builtin_amdgcn_make_buffer_rsrc(pb, 0, nr * N, 0x00020000);
    qs = __builtin_amdgcn_make_buffer_rsrc(ps, 0, nr * ns, 0x00020000);
    left -= BKR;
    pa += (int64_t)BKR * ld4; pb += (int64_t)BKR * N; ps += (int64_t)BKR * ns;
  };
  struct Regs { u32x4 a[4]; uint32_t b[4], s[4]; } R[2];
  auto load = [&](Regs& r, int i) {                        // row i of the thread's block
    r.a[i] = __builtin_amdgcn_raw_buffer_load_b128(qa, va + i * ld4, 0, 0);
    r.b[i] = __builtin_amdgcn_raw_buffer_load_b32(qb, vb + i * N, 0, 0);
    r.s[i] = __builtin_amdgcn_raw_buffer_load_b8(qs, vs + i * ns, 0, 0);
  };
  auto load_all = [&](Regs& r) {
    next_rows();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      load(r, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto store_a = [&](const Regs& r, int e, int buf) {      // column e of it
    la[buf][rg * BT + f32_place(c4 + e)] = u32x4{r.a[0][e], r.a[1][e], r.a[2][e], r.a[3][e]};
  };
  auto store_b = [&](const Regs& r, int e, int buf) {
    lb[buf][rg * BT + f32_place(c4 + e)] = f32x4{q8_code(r.b[0], e) * q8_scale(r.s[0]), q8_code(r.b[1], e) * q8_scale(r.s[1]),
                                                 q8_code(r.b[2], e) * q8_scale(r.s[2]), q8_code(r.b[3], e) * q8_scale(r.s[3])};
  };

  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  const int fa = (l >> 5) * BT + f32_place(wm), fb = (l >> 5) * BT + f32_place(wn);
  f32x4 A[2] = {}, B[2] = {};                              // fragments of eight rows: the lower half of the wave the first four
  // eight parts: products of eight rows, reads of the next eight; the first four parts also store the next step's rows, which have
  // waited in registers for a step, the last four load what takes their place (two steps on).  The order is the one written: a product, then what the matrix unit's 64 cycles leave room for
  auto step = [&](auto bufc) {
    constexpr int buf = decltype(bufc)::value;
    Regs& r = R[buf ^ 1];
    lds_barrier();
    next_rows();
    static_for<BKR / 8>([&](auto tc) {
      constexpr int t = decltype(tc)::value, cur = (t + 1) & 1, nxt = t & 1;
      static_for<4>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(A[cur][e], B[cur][e], acc, 0, 0, 0);
        if constexpr (e == 0) { A[nxt] = __builtin_bit_cast(f32x4, la[buf][fa + 2 * t * BT]); B[nxt] = lb[buf][fb + 2 * t * BT]; }
        if constexpr (e == 1 && t < 4) store_a(r, t, buf ^ 1);
        if constexpr (e == 2 && t < 4) store_b(r, t, buf ^ 1);
        if constexpr (e == 2 && t >= 4) load(r, t - 4);
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  if (k_beg < k_end) {
    load_all(R[0]);
    load_all(R[1]);
    __builtin_amdgcn_sched_barrier(0);                    // (the counted waits of the loop need R[1]'s loads in front of R[0]'s next ones)
#pragma unroll
    for (int e = 0; e < 4; ++e) { store_a(R[0], e, 0); store_b(R[0], e, 0); }
    load_all(R[0]);
    int k = k_beg + 1;
    for (; k < k_end; k += 2) {
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    }
    if (k == k_end) step(std::integral_constant<int, 0>{});
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(A[1][e], B[1][e], acc, 0, 0, 0);
  }

  const bool add = P.splits == 1 && args.accumulate;
  const int n = n0 + wn;
  if (n >= N) return;
  float* o = (P.splits == 1 ? P.out : P.slab + (int64_t)z * M * N) + n;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int m = m0 + (wave >> 1) * 32 + 8 * e + 4 * (l >> 5);
    if (m >= M) continue;                                  // (M is a multiple of 8)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float* q = o + (int64_t)(m + c) * N;
      *q = add ? *q + acc[4 * e + c] : acc[4 * e + c];
    }
  }
}

// ------------------------------------------------------------------------------------------------- bf16
// Tile (32 MI WM) x (32 NI WN), KG groups of WM x WN waves with MI x NI products of 32 x 32 x 16 each; 64 rows of dY and X a step and group,
// two buffers in LDS.  The groups take the lower and the upper rows of a step; their sums meet in LDS at the end.  KG = 2 serves the smallest
// tile, 64 x 64 with one product a wave, whose step is bound by what one wave can issue: 128 rows take 0.47 us, 64 rows with one group 0.31.
// dY goes to LDS without a stop in registers; codes wait about two steps in registers and become bf16 on their way to LDS.
//   barrier (step k's buffer is complete, the other one free)
//   part 0: products of step k - 1's last 16 rows, reads of the fragments of step k's rows 0 .. 15, loads of the dY of step k + 1
//   parts 1 - 3: products of 16 rows of step k, reads of the next 16
// Parts 0 - 2 also store a third each of step k + 1's X into the other buffer and load what takes its registers' place; part 3 reads
// early and stores nothing, so that nothing is left to wait for at the barrier, and the products behind the barrier have their
// fragments in registers.  Reads, conversions and loads stand between the products in the order written.
//
// Measured at 256 x 256: 1.21 us a step on part of the chip (70 % of the matrix rate at 2.4 GHz), 1.65 us with every CU at work, where
// the power of the matrix units lowers the clock to about 1.8 GHz: 4096 x 4096 over 16,384 rows take 421 us, 1,305 TFLOP/s; a large
// library product of bf16 matrices reaches 1,600 on this card, this kernel without its conversions and loads about 1,550.  No bank
// conflicts are counted.  Not faster: four waves with 128 x 128 each (1.38 us a step: a store blocks the wave that also has to feed the
// matrix unit), a third buffer of dY, the conversions spread over all four parts; touching dY's lines a step ahead costs 15 %.
//
// LDS image: [rows][columns] bf16, the 64-byte unit u of row r at u ^ (r & 3) (two units a row: u ^ (r >> 1 & 1)): the four rows x 64 bytes
// that half a wave reads in one transposing read lie in different banks, and so do the stores (served eight lanes at a time).

// four rows of 16 columns, transposed (all lanes of the wave take part)
__device__ __forceinline__ s16x4 tr_read(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
struct Frag8 {                                            // eight rows of a column: two transposed reads
  s16x4 h[2];
  __device__ __forceinline__ bf16x8 v() const {
    union { s16x4 s[2]; bf16x8 b; } u;
    u.s[0] = h[0]; u.s[1] = h[1];
    return u.b;
  }
};

// what the unit of a row is moved by; the lower two bits of the row decide
template <int COLS> __device__ __forceinline__ int place(int row) { return COLS >= 128 ? row & 3 : row >> 1 & 1; }

template <int MI, int NI, int WM, int WN, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void wgrad_bf16_kernel(const Args args) {
  constexpr int NW = WM * WN * KG, NT = 64 * NW, STEP = 64 * KG, TM = 32 * MI * WM, TN = 32 * NI * WN, RA = TM * 2, RB = TN * 2;
  constexpr int CA = TM / 8, CB = TN / 16;                // 16-byte chunks of a row of dY / of codes
  constexpr int NA = STEP * CA / NT, NB = STEP * CB / NT, DA = NT / CA, DB = NT / CB;      // chunks a thread, rows between them
  // one object a buffer: the compiler then sees that a read of one does not wait for what arrives in another
  __shared__ __attribute__((aligned(1024))) char A0[STEP * RA], A1[STEP * RA], B0[STEP * RB], B1[STEP * RB];

  const int w = work_of_block(args.p[args.count - 1].work_end);
  int which = 0;
  for (int i = 0; i < MAXP - 1; ++i) which += i < args.count - 1 && w >= args.p[i].work_end ? 1 : 0;
  const Problem& P = args.p[which];
  const int local = w - (which ? args.p[which - 1].work_end : 0);
  const int z = local / P.tiles, tile = local - z * P.tiles;
  const int m0 = tile / P.tiles_n * TM, n0 = tile % P.tiles_n * TN;
  const int k_beg = z * P.steps_per_split, k_end = min(k_beg + P.steps_per_split, P.steps);
  const int M = P.M, N = P.N;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
  const int kg = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;

  // ---- global side: chunk i of a thread is DA (DB) rows below chunk i - 1.  The resources cover the rows of the step, so rows behind
  // the range read as zero; columns outside are given an offset beyond every resource.  16 codes come as two loads of 8: four of each
  // eight lanes take (and store) the upper half first, so that the eight 16-byte stores served at once touch different banks
  const int ra = tid / CA, ua = (tid % CA >> 2) ^ place<TM>(ra), ca = 4 * ua + (tid & 3), rb = tid / CB, cb = tid % CB, hb = (tid >> 2) & 1;
  const int ld2 = (int)(P.lddy * 2), ns = N / ACTQ8_GROUP;
  const uint32_t va = m0 + 8 * ca < M ? ra * ld2 + (m0 + 8 * ca) * 2 : OUTSIDE;
  const uint32_t vb = n0 + 16 * cb < N ? rb * N + n0 + 16 * cb + 8 * hb : OUTSIDE, vb2 = second_half(vb, hb);
  const uint32_t vs = n0 + 16 * cb < N ? rb * ns + (n0 + 16 * cb) / ACTQ8_GROUP : OUTSIDE;
  struct Regs { u32x2 b[NB][2]; uint32_t s[NB]; } R[2];
  const int64_t r_beg = (int64_t)k_beg * STEP;
  int left = (int)(min(P.rows, (int64_t)k_end * STEP) - r_beg);
  int left_a = left;
  char* pa = (char*)P.dy + r_beg * ld2;
  char* pb = (char*)P.codes + r_beg * N;
  char* ps = (char*)P.scales + r_beg * ns;
  __amdgpu_buffer_rsrc_t qa, qb, qs;
  auto next_rows = [&]() {                                // the resources of the next step's rows (none left: empty ones)
    const int nr = __builtin_amdgcn_readfirstlane(max(min(left, STEP), 0));
    qb = __builtin_amdgcn_make_buffer_rsrc(pb, 0, nr * N, 0x00020000);
    qs = __builtin_amdgcn_make_buffer_rsrc(ps, 0, nr * ns, 0x00020000);
    left -= STEP;
    pb += (int64_t)STEP * N; ps += (int64_t)STEP * ns;
  };
  auto next_rows_a = [&]() {
    const int nr = __builtin_amdgcn_readfirstlane(max(min(left_a, STEP), 0));
    qa = __builtin_amdgcn_make_buffer_rsrc(pa, 0, nr * ld2, 0x00020000);
    left_a -= STEP;
    pa += (int64_t)STEP * ld2;
  };
  // a step's chunks of dY and half chunks of codes in three shares
  constexpr auto a_from = [](int t) { return (t * NA + 2) / 3; };
  constexpr auto b_from = [](int t) { return t * 2 * NB / 3; };
  // dY goes to LDS without a stop in registers: 64 lanes x 16 bytes in a row, so the unit's place is chosen on the source side
  auto load_a = [&](int i, auto bufc) {
    char* d = (decltype(bufc)::value ? A1 : A0) + (NW * i + wave) * 1024;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(qa, (__attribute__((address_space(3))) void*)d, 16, va + i * DA * ld2, 0, 0, 0);
  };
  auto load_b = [&](Regs& r, int i) {                     // half chunk i; the chunk's scale behind its second half
    r.b[i >> 1][i & 1] = __builtin_amdgcn_raw_buffer_load_b64(qb, ((i & 1) ? vb2 : vb) + (i >> 1) * DB * N, 0, 0);
    if (i & 1) r.s[i >> 1] = __builtin_amdgcn_raw_buffer_load_b8(qs, vs + (i >> 1) * DB * ns, 0, 0);
  };

  // ---- LDS side.  DA and DB are multiples of 4: a thread's rows agree in their lower two bits
  static_assert(DA % 4 == 0 && DB % 4 == 0, "the unit's place depends on the thread alone");
  const int ob = rb * RB + (((cb >> 1) ^ place<TN>(rb)) << 6) + (cb & 1) * 32 + 16 * hb, ob2 = ob + 16 - 32 * hb;
  u32x4 conv;                                             // the half chunk under conversion
  float cs = 0.f;                                         // and its scale
  auto convert = [&](const Regs& r, int i, int e, auto bufc) {                   // two codes of half chunk i; the last two store it
    if (e == 0) cs = q8_scale(r.s[i >> 1]);
    const uint32_t w = r.b[i >> 1][i & 1][e >> 1];
    conv[e] = pack_exact_bf16(q8_code(w, 2 * (e & 1)) * cs, q8_code(w, 2 * (e & 1) + 1) * cs);
    if (e == 3) *reinterpret_cast<u32x4*>((decltype(bufc)::value ? B1 : B0) + ((i & 1) ? ob2 : ob) + (i >> 1) * DB * RB) = conv;
  };

  // ---- fragments: lane (half, col & 31): 8 rows 8 half .. + 7 of a part.  A transposing read gives 16 lanes a 4 x 16 block
  const int g = l >> 4, q = (l >> 2) & 3, p4 = l & 3;
  int fa[MI], fb[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) fa[i] = (64 * kg + 8 * (g >> 1) + q) * RA + (((wm * MI + i) ^ place<TM>(q)) << 6) + (g & 1) * 32 + p4 * 8;
#pragma unroll
  for (int j = 0; j < NI; ++j) fb[j] = (64 * kg + 8 * (g >> 1) + q) * RB + (((wn * NI + j) ^ place<TN>(q)) << 6) + (g & 1) * 32 + p4 * 8;
  struct Frags { Frag8 a[MI], b[NI]; } F[2];
  auto read = [&](Frags& f, int i, auto bufc, int part) { // read i of 2 (NI + MI)
    const int row = part * 16 + 4 * (i & 1);
    if (i < 2 * NI) f.b[i >> 1].h[i & 1] = tr_read((decltype(bufc)::value ? B1 : B0) + fb[i >> 1] + row * RB);
    else f.a[(i >> 1) - NI].h[i & 1] = tr_read((decltype(bufc)::value ? A1 : A0) + fa[(i >> 1) - NI] + row * RA);
  };
  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  auto mma = [&](const Frags& f, int i) {
    acc[i / NI][i % NI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a[i / NI].v(), f.b[i % NI].v(), acc[i / NI][i % NI], 0, 0, 0);
  };
  // vector loads of a step behind its loads of dY: the half chunks of shares 1 and 2 and their scales at least
  constexpr int BEHIND = (2 * NB - b_from(1)) + (NB - b_from(1) / 2);
  constexpr int WAIT = (BEHIND & 15) | (BEHIND >> 4 << 14) | (7 << 4) | (15 << 8);       // vmcnt(BEHIND), the other counters free
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  // one part: products of f, fragments of (buffer rbuf, part rpart) to n; share T < 3 of r to buffer sbuf, its registers refilled.  The
  // order is the one written here: a product, then what the matrix unit's 32 cycles leave room for
  auto part = [&](const Frags& f, Frags& n, auto rbuf, int rpart, Regs& r, auto tc, auto sbuf) {
    constexpr int T = decltype(tc)::value, P = MI * NI, RD = 2 * (MI + NI), RP = T < 3 || P == 1 ? P : P / 2;
    constexpr int na = T == 0 ? NA : 0, b0 = T < 3 ? b_from(T) : 0, nc = T < 3 ? 4 * (b_from(T + 1) - b0) : 0;
    static_for<P>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      mma(f, i);
#pragma unroll
      for (int k = std::min(i, RP) * RD / RP; k < std::min(i + 1, RP) * RD / RP; ++k) read(n, k, rbuf, rpart);
#pragma unroll
      for (int k = i * na / P; k < (i + 1) * na / P; ++k) load_a(k, sbuf);
#pragma unroll
      for (int k = i * nc / P; k < (i + 1) * nc / P; ++k) {
        convert(r, b0 + k / 4, k % 4, sbuf);
        if (k % 4 == 3) load_b(r, b0 + k / 4);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto step = [&](auto bufc) {
    constexpr int b = decltype(bufc)::value;
    using Cur = std::integral_constant<int, b>;
    using Oth = std::integral_constant<int, b ^ 1>;
    Regs& r = R[b ^ 1];
    __builtin_amdgcn_s_waitcnt(WAIT);                     // this wave's dY of the step has arrived (the loads of codes behind it need not have)
    lds_barrier();
    next_rows();
    next_rows_a();
    part(F[1], F[0], Cur{}, 0, r, I0{}, Oth{});
    part(F[0], F[1], Cur{}, 1, r, I1{}, Oth{});
    part(F[1], F[0], Cur{}, 2, r, I2{}, Oth{});
    part(F[0], F[1], Cur{}, 3, r, I3{}, Oth{});
  };

  if (k_beg < k_end) {
    auto load_all = [&](Regs& r) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) load_b(r, i);
    };
    next_rows_a();
#pragma unroll
    for (int i = 0; i < NA; ++i) load_a(i, I0{});
    next_rows();
    load_all(R[0]);
    next_rows();
    load_all(R[1]);
#pragma unroll
    for (int i = 0; i < 8 * NB; ++i) convert(R[0], i / 4, i % 4, I0{});
    next_rows();
    load_all(R[0]);
#pragma unroll
    for (int i = 0; i < MI; ++i) F[1].a[i] = Frag8{};
#pragma unroll
    for (int j = 0; j < NI; ++j) F[1].b[j] = Frag8{};
    if constexpr (KG == 1) {
      for (int k = k_beg; k < k_end; k += 2) {            // (behind the last step of an odd range: one on zeros)
        step(I0{});
        step(I1{});
      }
    } else {
      int k = k_beg + 1;
      for (; k < k_end; k += 2) {
        step(I0{});
        step(I1{});
      }
      if (k == k_end) step(I0{});
    }
#pragma unroll
    for (int i = 0; i < MI * NI; ++i) mma(F[1], i);
    __builtin_amdgcn_s_waitcnt(15 << 8 | 7 << 4);           // nothing arrives in LDS behind the wave's end: vmcnt(0)
  }
  if constexpr (KG == 2) {                                // the upper rows' sums join the lower rows'
    static_assert(MI * NI == 1 && STEP * RA >= 4 * 64 * WM * WN * 16, "a wave's sums fit its share of a buffer");
    f32x4* s = reinterpret_cast<f32x4*>(A0) + (wave % (WM * WN)) * 256 + l;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (kg == 1) s[e * 64] = f32x4{acc[0][0][4 * e], acc[0][0][4 * e + 1], acc[0][0][4 * e + 2], acc[0][0][4 * e + 3]};
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x4 v = s[e * 64];
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[0][0][4 * e + c] += v[c];
    }
  }

  // ---- sums: to the slab in the order of the registers (16 bytes a lane, whole lines), or to their places
  if (P.splits > 1) {
    f32x4* s = reinterpret_cast<f32x4*>(P.slab) + ((int64_t)(z * P.tiles + tile) * (TM * TN / 4)) + wave * (MI * NI * 4 * 64) + l;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f32x4 v;
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = acc[i][j][4 * e + c];
          s[((i * NI + j) * 4 + e) * 64] = v;
        }
    return;
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = n0 + (wn * NI + j) * 32 + (l & 31);
      if (n >= N) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + (wm * MI + i) * 32 + 8 * e + 4 * (l >> 5);
        if (m >= M) continue;                             // (M is a multiple of 8)
        float* o = P.out + (int64_t)m * N + n;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[(int64_t)c * N] = args.accumulate ? o[(int64_t)c * N] + acc[i][j][4 * e + c] : acc[i][j][4 * e + c];
      }
    }
}

// out (+)= the slabs of wgrad_bf16_kernel in the order of the row ranges; a block takes one (i, j) product of a wave: 256 f32x4 a slab
template <int MI, int NI, int WM, int WN>
__global__ __launch_bounds__(256) void wgrad_join_bf16_kernel(const Args args) {
  constexpr int PER = WM * WN * MI * NI;                  // blocks a tile
  const int l = threadIdx.x & 63, e = threadIdx.x >> 6;
  int b = blockIdx.x, which = 0;
  for (; which < args.count; ++which) {
    const int mine = args.p[which].splits > 1 ? args.p[which].tiles * PER : 0;
    if (b < mine) break;
    b -= mine;
  }
  const Problem& P = args.p[which];
  const int tile = b / PER, sub = b % PER, wave = sub / (MI * NI), ij = sub % (MI * NI);
  const int n = tile % P.tiles_n * (32 * NI * WN) + (wave % WN * NI + ij % NI) * 32 + (l & 31);
  const int m = tile / P.tiles_n * (32 * MI * WM) + (wave / WN * MI + ij / NI) * 32 + 8 * e + 4 * (l >> 5);
  if (n >= P.N || m >= P.M) return;
  const f32x4* s = reinterpret_cast<const f32x4*>(P.slab) + ((int64_t)tile * PER + sub) * 256 + threadIdx.x;
  const int64_t stride = (int64_t)P.tiles * PER * 256;
  f32x4 v = s[0];
#pragma unroll 4
  for (int z = 1; z < P.splits; ++z) v += s[z * stride];
  float* o = P.out + (int64_t)m * P.N + n;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[(int64_t)c * P.N] = args.accumulate ? o[(int64_t)c * P.N] + v[c] : v[c];
}

// out (+)= the slabs of wgrad_f32_kernel in the order of the row ranges
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

// Tile variants and the number of row ranges.  Time of a step with one tile on the chip's CUs or fewer (`one`) and with every place taken
// (`full`: the clock drops with the power that the matrix units draw; between them in proportion, for the smallest tile at once when two
// of its blocks share a CU), measured on 2304 x 768, 4096 x 4096 and, the smallest, 768 x 768 and 2304 x 768; a range costs about 3 us to
// start and end, a join 4 us and 5.5 TB/s for writing and reading the slabs.  Over 34 sets of sizes from 192 x 192 to a layer of 1024 / 4096,
// 130 to 34,000 rows, each timed with every tile and 16 numbers of ranges, the choice is 1 % off the best on average and 15 % at most.  The large tile moves the fewest bytes per product, the
// small ones fill the chip on small outputs with fewer ranges, hence smaller slabs: 768 x 768 over 1,025 rows takes 7.8 us with the smallest
// tile and no range, 12.7 us with 128 x 128 in two.
struct Variant { int tm, tn, step, slots; double one, full; };
constexpr Variant VAR[4] = {{256, 256, 64, 256, 1.21, 1.65}, {256, 128, 64, 256, 0.76, 0.97}, {128, 128, 64, 512, 0.58, 1.11}, {64, 64, 128, 512, 0.50, 0.87}};

// sets tiles, row ranges and work of the problems for (tile, at most s ranges); returns the bytes of slabs
int64_t lay_out(Args& a, int tm, int tn, int step, int s, bool exact_slabs) {
  int64_t bytes = 0, work = 0;
  for (int i = 0; i < a.count; ++i) {
    Problem& p = a.p[i];
    p.tiles_n = ceil_div(p.N, tn);
    p.tiles = ceil_div(p.M, tm) * p.tiles_n;
    p.steps = ceil_div(p.rows, step);
    p.steps_per_split = ceil_div(p.steps, std::max(1, std::min(s, p.steps / 2)));
    p.splits = ceil_div(p.steps, p.steps_per_split);
    work += (int64_t)p.tiles * p.splits;
    p.work_end = (int)std::min<int64_t>(work, INT32_MAX);
    if (p.splits > 1) {
      p.slab = reinterpret_cast<float*>(bytes);            // offset, resolved against the workspace by the caller
      bytes += (int64_t)p.splits * (exact_slabs ? (int64_t)p.M * p.N : (int64_t)p.tiles * tm * tn) * 4;
    }
  }
  return bytes;
}

// chooses the tile and the row ranges of the problems; returns the bytes of slabs, or -1
int64_t plan(Args& a, int dtype) {
  for (int i = 0; i < a.count; ++i) {
    const Problem& p = a.p[i];
    if (p.M <= 0 || p.N <= 0 || p.rows <= 0 || p.M % 8 || p.N % ACTQ8_GROUP || p.rows >= (1LL << 31) - 128 || (int64_t)p.M * p.N > (1LL << 31)) return -1;
  }
  if (dtype == S4F_F32) {
    // as many ranges as give every CU one, two .. twelve blocks, by the time of a step of 64 rows: 1.17 us with one block on a CU, 1.05 for
    // each of several; start, end, join and slabs as below (520 x 416 over 2,307 rows: 19 us with 4 ranges of 10 steps, 21 with 8 of 5; 768 x 768
    // over 16,400: 164 us with 7, 186 with 3)
    lay_out(a, BT, BT, BKR, 1, true);
    const int tiles = a.p[a.count - 1].work_end;
    double best = 0;
    int bs = 1, last = 0;
    for (int c = 0; c <= 12; ++c) {
      const int s = std::max(1, 256 * c / tiles);
      if (s == last) continue;
      last = s;
      int64_t items = 0, slabs = 0;
      int longest = 0;
      for (int i = 0; i < a.count; ++i) {
        const int each = ceil_div(a.p[i].steps, std::max(1, std::min(s, a.p[i].steps / 2))), n = ceil_div(a.p[i].steps, each);
        longest = std::max(longest, each);
        items += (int64_t)a.p[i].tiles * n;
        if (n > 1) slabs += (int64_t)a.p[i].M * a.p[i].N * n;
      }
      const int64_t share = (items + 255) / 256;
      const double t = longest * (share == 1 ? 1.17 : 1.05 * share) + 3 + (slabs ? 4 + 8e-6 / 5.5 * slabs : 0);
      if (c == 0 || t < best) { best = t; bs = s; }
    }
    const int64_t bytes = lay_out(a, BT, BT, BKR, bs, true);
    return a.p[a.count - 1].work_end < INT32_MAX ? bytes : -1;
  }
  double best = 0;
  int bs = 0;
  for (int v = 0; v < 4; ++v) {
    int64_t tiles[MAXP], all = 0;
    for (int i = 0; i < a.count; ++i) {
      tiles[i] = (int64_t)ceil_div(a.p[i].M, VAR[v].tm) * ceil_div(a.p[i].N, VAR[v].tn);
      all += tiles[i];
    }
    const int most = (int)std::min<int64_t>(VAR[v].slots / all, 64);             // ranges that take every place once
    for (int s : {1, 2, 3, 4, most / 2, most}) {
      if (s < 1) continue;
      int64_t items = 0, slabs = 0;
      int longest = 0;
      for (int i = 0; i < a.count; ++i) {
        const int steps = ceil_div(a.p[i].rows, VAR[v].step), each = ceil_div(steps, std::max(1, std::min(s, steps / 2))), n = ceil_div(steps, each);
        longest = std::max(longest, each);
        items += tiles[i] * n;
        if (n > 1) slabs += tiles[i] * n;
      }
      const bool small = VAR[v].step == 128;
      const double rest = (double)(items % VAR[v].slots) / VAR[v].slots, fill = small ? rest > 0.5 : rest, per = (small ? longest : (longest + 1) & ~1) + 0.25;
      const double t = (double)(items / VAR[v].slots) * (per * VAR[v].full + 3) +
                       (rest > 0 ? per * (VAR[v].one + fill * (VAR[v].full - VAR[v].one)) + 3 : 0) +
                       (slabs ? 4 + 8e-6 / 5.5 * slabs * VAR[v].tm * VAR[v].tn : 0);
      if (bs == 0 || t < best) { best = t; a.variant = v; bs = s; }
    }
  }
  const int64_t bytes = lay_out(a, VAR[a.variant].tm, VAR[a.variant].tn, VAR[a.variant].step, bs, false);
  return a.p[a.count - 1].work_end < INT32_MAX ? bytes : -1;
}

template <int MI, int NI, int WM, int WN, int KG = 1> void launch_bf16(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL((wgrad_bf16_kernel<MI, NI, WM, WN, KG>), dim3(a.p[a.count - 1].work_end), dim3(64 * WM * WN * KG), 0, st, a);
  int blocks = 0;
  for (int i = 0; i < a.count; ++i) blocks += a.p[i].splits > 1 ? a.p[i].tiles * WM * WN * MI * NI : 0;
  if (blocks) hipLaunchKernelGGL((wgrad_join_bf16_kernel<MI, NI, WM, WN>), dim3(blocks), dim3(256), 0, st, a);
}

}  // namespace

// dims: {dtype, then M, N, rows of each problem}
int64_t s4f_wgrad_packed_ws(const int64_t* dims, int ndims) {
  if (ndims < 4 || (dims[0] != S4F_F32 && dims[0] != S4F_BF16) || (ndims - 1) % 3 || (ndims - 1) / 3 > MAXP) return -1;
  Args a{};
  a.count = (ndims - 1) / 3;
  for (int i = 0; i < a.count; ++i) {
    const int64_t* d = dims + 1 + 3 * i;
    if (d[0] <= 0 || d[0] > INT32_MAX || d[1] <= 0 || d[1] > INT32_MAX) return -1;
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
    S4F_CHECK((uintptr_t)d.dy % 16 == 0 && (uintptr_t)d.codes % 16 == 0 && (uintptr_t)d.out % 16 == 0 && d.lddy % (dtype == S4F_BF16 ? 8 : 4) == 0,
              "%s: rows of dy, codes and out must start on 16-byte boundaries (problem %d)", who, i);
    S4F_CHECK(d.M > 0 && d.N > 0 && d.rows > 0 && d.M % 8 == 0 && d.N % ACTQ8_GROUP == 0,
              "%s: M=%d must be a multiple of 8, N=%d of 32, rows=%lld positive", who, d.M, d.N, (long long)d.rows);
    S4F_CHECK(d.lddy >= d.M, "%s: rows of dy overlap (ld %lld < M %d)", who, (long long)d.lddy, d.M);
    // (the kernels address the rows of a step, 64 or 128, with offsets below 2^31)
    S4F_CHECK(d.lddy < (1 << 22) && d.N < (1 << 23) && d.rows < (1LL << 31) - 128, "%s: sizes too large for one launch", who);
    Problem& p = a.p[i];
    p.dy = d.dy; p.lddy = d.lddy; p.codes = d.codes; p.scales = d.scales; p.out = d.out; p.M = d.M; p.N = d.N; p.rows = d.rows;
  }
  const int64_t need = plan(a, dtype);
  S4F_CHECK(need >= 0, "%s: sizes too large for one launch", who);
  S4F_CHECK(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need), "%s: workspace missing, misaligned or too small (%lld < %lld)",
            who, (long long)ws_bytes, (long long)need);
  for (int i = 0; i < count; ++i) {
    const Problem& p = a.p[i];
    const Piece out = piece(p.out, (int64_t)p.M * p.N * 4), slabs = piece(ws, ws_bytes);
    bool bad = meet(out, slabs);
    for (int j = 0; j < count; ++j) {
      const Problem& o = a.p[j];
      const Piece dy = piece(o.dy, o.rows, o.lddy, o.M, dtype == S4F_BF16 ? 2 : 4), c = piece(o.codes, o.rows * o.N),
                  s = piece(o.scales, o.rows * (o.N / ACTQ8_GROUP));
      bad = bad || meet(out, {dy, c, s}) || meet(slabs, {dy, c, s}) || (j != i && meet(out, piece(o.out, (int64_t)o.M * o.N * 4)));
    }
    S4F_CHECK(!bad, "%s: an output or the workspace overlaps another or an input (problem %d)", who, i);
  }
  bool join = false;
  int64_t n4 = 0;
  for (int i = 0; i < count; ++i)
    if (a.p[i].splits > 1) {
      a.p[i].slab = reinterpret_cast<float*>((char*)ws + (int64_t)reinterpret_cast<uintptr_t>(a.p[i].slab));
      join = true;
      n4 = std::max<int64_t>(n4, (int64_t)a.p[i].M * a.p[i].N / 4);
    }
  if (dtype == S4F_BF16) {
    if (a.variant == 0) launch_bf16<4, 2, 2, 4>(a, (hipStream_t)stream);
    else if (a.variant == 1) launch_bf16<2, 2, 4, 2>(a, (hipStream_t)stream);
    else if (a.variant == 2) launch_bf16<2, 2, 2, 2>(a, (hipStream_t)stream);
    else launch_bf16<1, 1, 2, 2, 2>(a, (hipStream_t)stream);
    S4F_LAUNCH_CHECK();
    return 0;
  }
  const dim3 grid(a.p[count - 1].work_end);
  hipLaunchKernelGGL(wgrad_f32_kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  S4F_LAUNCH_CHECK();
  if (join) {
    hipLaunchKernelGGL(wgrad_join_kernel, dim3((unsigned)std::min<int64_t>((n4 + 255) / 256, 2048)), dim3(256), 0, (hipStream_t)stream, a);
    S4F_LAUNCH_CHECK();
  }
  return 0;
}
