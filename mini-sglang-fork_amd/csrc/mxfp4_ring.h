// MXFP4 tile ring: BM x BN output tiles whose operands stream through LDS.
//
// y[m, n] = sum over blocks b of 2^(ea[m, b] + ew[n, b]) sum_i a[m, 32 b + i]
// w[n, 32 b + i]: v_mfma_scale_f32_32x32x64_f8f6f4 multiplies two blocks of 32
// rows and columns and applies both scales; sums are fp32.  With both operands in
// registers the instruction runs at 9.9 PFLOP/s on zeros and 6.7 on random
// codes (power); the 16x16x128 form reaches 6.9 and 5.5.
//
// Why this form: codes move by DMA from global memory into LDS (stages of 128
// bytes a row, the line size), so no register holds data in flight; 256 x 256
// tiles of 8 waves of 64 x 128 read 48 KB of LDS per 64 elements of K and CU
// beside 256 matrix cycles per SIMD pair; one block per CU walks its tiles, the
// first stages of the next one in flight during the epilogue; the weight rows
// are the instruction's rows, so that a lane holds 4 adjacent columns and the
// epilogue packs and stores from registers.  MI355X: 8192 x 34816 x 5120 691-735
// us (4.0-4.2 PFLOP/s), 8192 x 5120 x 17408 332 us (4.4).  What bounds it: without
// the DMA the first takes 556 us, with the DMA's lines in the L2 666 (a stage's
// loads have one stage to arrive; the LDS has no room for a third slot), and
// the output's stores the rest.
#pragma once

#include "gemm_kernels.h"
#include "mxfp4.h"

namespace mw8 {

// n / d for n < 2^31 as one multiplication: with 2^(l-1) < d <= 2^l and m =
// ceil(2^(31+l) / d) < 2^32 the excess m d - 2^(31+l) is below 2^l, so n m /
// 2^(31+l) stays below the next integer.  (A division by a runtime value
// runs as some 40 vector instructions; tiles are found between two tiles'
// matrix instructions.)
struct MxDivisor {
  uint32_t m, shift;
  static MxDivisor of(uint32_t d) {
    uint32_t l = 0;
    while ((1u << l) < d) ++l;
    return {static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), 31 + l};
  }
  MW8_HD uint32_t div(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift); }
};

// Tile order: tiles of a grid of tiles_m x tiles_n in groups of 4 tile rows
// that advance along N together; XCD b % 8 owns a contiguous range of them
// and starts x / 8 of the way in (as tile_of_block does for the int8 rings).
struct MxRaster {
  uint32_t tiles_m, tiles_n, count;
  MxDivisor group, last;  // by 4 tiles_n, and by the rows of a last short group
  static MxRaster of(int64_t m, int64_t n) {
    const uint32_t tm = static_cast<uint32_t>(m), tn = static_cast<uint32_t>(n);
    return {tm, tn, tm * tn, MxDivisor::of(4 * tn), MxDivisor::of(tm % 4 ? tm % 4 : 4)};
  }
  MW8_HD void tile(uint32_t b, uint32_t& pm, uint32_t& pn) const {
    const uint32_t xcd = b % 8, local = b / 8, base = count / 8, rem = count % 8;
    const uint32_t n_x = base + (xcd < rem ? 1 : 0), start = xcd * base + (xcd < rem ? xcd : rem);
    uint32_t at = local + xcd * (n_x / 8);
    if (at >= n_x) at -= n_x;
    const uint32_t t = start + at, g = group.div(t), in = t - g * 4 * tiles_n;
    const bool full = 4 * g + 4 <= tiles_m;
    const uint32_t rows = full ? 4 : tiles_m - 4 * g, col = full ? in >> 2 : last.div(in);
    pm = 4 * g + in - col * rows;
    pn = col;
  }
};

struct MxArgs {
  const uint8_t* A;   // codes [M, 16 kb]
  const uint8_t* sa;  // scales [tiles, M, 16]
  const uint8_t* W;   // codes [N, 16 kb]
  const uint8_t* sw;  // scales [tiles, N, 16]
  const uint16_t* bias;
  uint16_t* out;
  int64_t M, N;
  int kb;        // blocks of 32 along K
  int tiles;     // 512-element tiles along K
  int store;     // columns per output store: 8 (N % 8 == 0, out 16-byte aligned), 4 (N % 4 == 0, 8-byte) or 1
  MxRaster raster;
  // K split (kSplit kernels): grid count x split, block b takes the
  // 512-element tiles [tiles p / split, tiles (p + 1) / split) of output tile
  // b % count, p = b / count, and writes fp32 sums to part[p][M][N]
  float* part;
  int split;
  // long walks: blocks start in four groups, a quarter of a tile apart (units
  // of 2048 clocks)
  int stagger;
  // kAct kernels: W [2 I, K] holds gate rows, then up rows (N = 2 I); the output
  // is the quantized activation [M, I]
  uint8_t* q;
  uint8_t* s;
};

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

#if defined(__HIP_DEVICE_COMPILE__)
// D += W A over 128 elements of K, weight rows as the instruction's rows:
// lane l holds output columns (weight rows) 4 (l / 16) + v of token l % 16.
// J: the byte of the scale dwords.
template <int J>
__device__ __forceinline__ v4f mx_mma(v4i w, v4i a, v4f c, int sw, int sa) {
  const v8i x = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, y = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4 /* e2m1 */, 4, J, sw, J, sa);
}

// D += W A over 64 elements of K on 32 x 32: lane l holds columns (weight
// rows) 8 (v / 4) + 4 (l / 32) + v % 4 of token l % 32.
template <int J>
__device__ __forceinline__ v16f mx_mma32(v4i w, v4i a, v16f c, int sw, int sa) {
  const v8i x = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, y = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4 /* e2m1 */, 4, J, sw, J, sa);
}
#endif

// Stages of 256 K elements (128 bytes a row), NS data slots; the scales of
// 512 elements (16 bytes a row) come with every even stage.
template <int BM, int BN, int WM, int WN, int NS>
struct MxRing {
  static constexpr int kWaves = WM * WN;
  static constexpr int kStageA = BM * 128, kStageB = BN * 128, kStage = kStageA + kStageB;
  static constexpr int kScaleSlots = (NS + 1) / 2;
  static constexpr int kScale = (BM + BN) * 16;
  static constexpr int kLds = NS * kStage + kScaleSlots * kScale;
};

// kAct >= 0 (the activation's code): the tile's weight rows are BN / 2 gate
// rows and the matching up rows, so that a wave holds both of a column (its
// first half of fragments gate, its second up).  The epilogue rounds both
// to bf16, as the plain product stores them, and writes the MXFP4 codes and
// scales of bf16(act(gate) up): a 32-column fragment is one block per row,
// shared by lanes l and l + 32.
template <int BM, int BN, int WM, int WN, int NS, bool kSplit, int kAct>
__global__ __launch_bounds__(64 * WM * WN) void mxfp4_ring_kernel(MxArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using R = MxRing<BM, BN, WM, WN, NS>;
  constexpr int kWaves = R::kWaves;
  constexpr int kWaveM = BM / WM, kWaveN = BN / WN;
  constexpr int kFM = kWaveM / 32, kFN = kWaveN / 32;
  constexpr int kLA = BM / (8 * kWaves), kLB = BN / (8 * kWaves);
  constexpr int kL = kLA + kLB;                          // data DMA instructions per wave and stage
  constexpr int kSUnits = (BM + BN) / 64;                // scale DMA instructions per 512 elements
  constexpr int kLS = (kSUnits + kWaves - 1) / kWaves;   // per wave (the last repeated where it does not divide)
  constexpr int kStores = kAct >= 0 ? kFM * kFN : kFM * kFN * 2;  // store instructions per wave and tile
  constexpr int kTileN = kAct >= 0 ? BN / 2 : BN;        // output columns of a tile
  constexpr int kHalf = kWaveN / 2;                      // kAct: gate rows of a wave, and up rows
  constexpr bool kWalk = NS == 2;                        // a block walks tiles blockIdx, blockIdx + gridDim, ...
  static_assert(kLA * 8 * kWaves == BM && kLB * 8 * kWaves == BN && BM % 64 == 0 && BN % 64 == 0, "DMA split");
  static_assert(!kSplit || !kWalk, "a split block owns one tile");
  static_assert(kAct < 0 || (!kSplit && kHalf == 64), "fused activation: a scale instruction loads one half");
  const int64_t inter = g.N / 2;  // kAct: rows of each half of W
  static_assert(NS >= 2 && NS <= 4 && R::kLds <= 163840 && kStores + kL + kLS < 64, "ring");
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int r32 = lane & 31, grp = lane >> 5;
  const uint32_t count = g.raster.count;
  const int64_t ld = static_cast<int64_t>(g.kb) * 16;
  const uint32_t kpart = kSplit ? blockIdx.x / count : 0;
  const int kt0 = kSplit ? static_cast<int>(static_cast<int64_t>(g.tiles) * kpart / g.split) : 0;
  const int kt1 = kSplit ? static_cast<int>(static_cast<int64_t>(g.tiles) * (kpart + 1) / g.split) : g.tiles;
  const int ns = 2 * (kt1 - kt0);  // stages; the second of the last 512 elements may be past K

  // The operands of one output tile.  Buffer views of its rows: bytes past
  // the last row read as zeros; those past a row's end read the next row's
  // (their scale bytes are 0 on both sides: the products vanish).
  // Scale instruction j of this wave fills rows 64 u .. 64 u + 63 of the slot
  // (the tile's A rows, then its W rows), u = j kWaves + wave; the last is
  // repeated where waves are left over.
  struct Tile {
    int64_t m0, n0;
    const uint8_t *a, *w;
    int rows_m, rows_n;  // 0: no tile, every load reads zeros
    const uint8_t* s[kLS];
    int s_bytes[kLS];
  };
  int64_t s_step[kLS];  // bytes from one 512 elements' scales to the next
#pragma unroll
  for (int j = 0; j < kLS; ++j) {
    const int u = j * kWaves + wave < kSUnits ? j * kWaves + wave : kSUnits - 1;
    s_step[j] = (u < BM / 64 ? g.M : g.N) * 16;
  }
  auto tile_at = [&](uint32_t t) {
    Tile o;
    uint32_t pm, pn;
    const bool live = t < count;
    g.raster.tile(live ? t : 0, pm, pn);
    o.m0 = static_cast<int64_t>(pm) * BM;
    o.n0 = static_cast<int64_t>(pn) * kTileN;
    o.a = g.A + o.m0 * ld;
    o.w = g.W + o.n0 * ld;
    o.rows_m = live ? static_cast<int>(g.M - o.m0 < BM ? g.M - o.m0 : BM) : 0;
    // (kAct: every row from the tile's first on, the up rows lie I further)
    o.rows_n = !live ? 0 : static_cast<int>(kAct >= 0 || g.N - o.n0 < BN ? g.N - o.n0 : BN);
#pragma unroll
    for (int j = 0; j < kLS; ++j) {
      const int u = j * kWaves + wave < kSUnits ? j * kWaves + wave : kSUnits - 1, uw = u - BM / 64;
      const bool is_a = uw < 0;
      int64_t row = is_a ? u * 64 : uw * 64;
      if constexpr (kAct >= 0) row = is_a ? u * 64 : (uw >> 1) * kHalf + (uw & 1) * inter;
      const int64_t left = (is_a ? o.rows_m : o.rows_n) - row;
      o.s[j] = (is_a ? g.sa + (kt0 * g.M + o.m0) * 16 : g.sw + (kt0 * g.N + o.n0) * 16) + row * 16;
      o.s_bytes[j] = __builtin_amdgcn_readfirstlane(static_cast<int>(left < 0 ? 0 : left < 64 ? left * 16 : 1024));
    }
    return o;
  };
  // field by field (a choice between two references would put both in memory)
  auto pick = [](bool c, const Tile& x, const Tile& y) {
    Tile o{c ? x.m0 : y.m0, c ? x.n0 : y.n0, c ? x.a : y.a, c ? x.w : y.w, c ? x.rows_m : y.rows_m, c ? x.rows_n : y.rows_n, {}, {}};
#pragma unroll
    for (int j = 0; j < kLS; ++j) {
      o.s[j] = c ? x.s[j] : y.s[j];
      o.s_bytes[j] = c ? x.s_bytes[j] : y.s_bytes[j];
    }
    return o;
  };
  auto view = [](const uint8_t* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(scalar_ptr(const_cast<uint8_t*>(p)), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kBufferFlags);
  };
  // LDS unit of a lane -> row and 16-byte chunk of the tile
  uint32_t a_off[kLA], w_off[kLB];
#pragma unroll
  for (int j = 0; j < kLA; ++j) {
    const int unit = (j * kWaves + wave) * 64 + lane, row = unit >> 3;
    a_off[j] = static_cast<uint32_t>(row * ld + 16 * ((unit & 7) ^ swz_f<128>(row)));
  }
#pragma unroll
  for (int j = 0; j < kLB; ++j) {
    const int unit = (j * kWaves + wave) * 64 + lane, row = unit >> 3;
    int64_t at = row;  // the tile row's row of W from the tile's first
    if constexpr (kAct >= 0) at = row / kWaveN * kHalf + row % kHalf + (row % kWaveN < kHalf ? 0 : inter);
    w_off[j] = static_cast<uint32_t>(at * ld + 16 * ((unit & 7) ^ swz_f<128>(row)));
  }
  auto issue_data = [&](const Tile& o, int slot, int s) {
    unsigned char* base = lds + slot * R::kStage;
    const __amdgpu_buffer_rsrc_t ra = view(o.a, o.rows_m * ld), rw = view(o.w, o.rows_n * ld);
    const int k0 = kt0 * 256 + s * 128;
#pragma unroll
    for (int j = 0; j < kLA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(base + (j * kWaves + wave) * 1024), 16, a_off[j], k0, 0, 0);
#pragma unroll
    for (int j = 0; j < kLB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr_t)(base + R::kStageA + (j * kWaves + wave) * 1024), 16, w_off[j],
                                               k0, 0, 0);
  };
  // scales of the tile's 512 elements number p
  auto issue_scales = [&](const Tile& o, int slot, int p) {
    unsigned char* base = lds + NS * R::kStage + slot * R::kScale;
#pragma unroll
    for (int j = 0; j < kLS; ++j) {
      const int u = j * kWaves + wave < kSUnits ? j * kWaves + wave : kSUnits - 1;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(view(o.s[j] + p * s_step[j], o.s_bytes[j]), (lds_ptr_t)(base + u * 1024), 16,
                                               lane * 16, 0, 0, 0);
    }
  };

  // Fragments: lane group g (l / 32) multiplies chunk 4 h + 2 g + u of a
  // stage in step 2 h + u; its scales of the stages of a tile are bytes
  // 2 t + u of the row's dwords g (h = 0) and g + 2 (h = 1).  The swizzle
  // depends on the row modulo 16 only, so a lane's fragments sit 32 rows apart.
  v4i fa[2][kFM], fb[2][kFN];
  int sa[kFM][2], sb[kFN][2];
  v16f acc[kFM][kFN];
  const int f_off = swz_lds<128>(r32, 2 * grp), s_off = r32 * 16 + 4 * grp;
  const unsigned char* const a_lds = lds + wm * kWaveM * 128;
  const unsigned char* const b_lds = lds + R::kStageA + wn * kWaveN * 128;
  const unsigned char* const sa_lds = lds + NS * R::kStage + wm * kWaveM * 16 + s_off;
  const unsigned char* const sb_lds = lds + NS * R::kStage + (BM + wn * kWaveN) * 16 + s_off;
  auto read_step = [&](int slot, int step) {
    const int off = slot * R::kStage + (f_off ^ ((step >> 1) * 64 + (step & 1) * 16));
#pragma unroll
    for (int j = 0; j < kFN; ++j) fb[step & 1][j] = *reinterpret_cast<const v4i*>(b_lds + off + j * 4096);
#pragma unroll
    for (int i = 0; i < kFM; ++i) fa[step & 1][i] = *reinterpret_cast<const v4i*>(a_lds + off + i * 4096);
  };
  auto read_scales = [&](int slot) {
    const int off = slot * R::kScale;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < kFN; ++j) sb[j][h] = *reinterpret_cast<const int*>(sb_lds + off + j * 512 + 8 * h);
#pragma unroll
      for (int i = 0; i < kFM; ++i) sa[i][h] = *reinterpret_cast<const int*>(sa_lds + off + i * 512 + 8 * h);
    }
  };
  auto mma_step = [&](auto pc, auto kc) {
    constexpr int J = 2 * decltype(pc)::value + (decltype(kc)::value & 1), h = decltype(kc)::value >> 1, set = decltype(kc)::value & 1;
#pragma unroll
    for (int j = 0; j < kFN; ++j)
#pragma unroll
      for (int i = 0; i < kFM; ++i) acc[i][j] = mx_mma32<J>(fb[set][j], fa[set][i], acc[i][j], sb[j][h], sa[i][h]);
  };
  // a step's reads go out one behind each of its first matrix instructions,
  // and stay in their step (moved further ahead they would need a third set of registers)
  auto phase_end = [] {
#pragma unroll
    for (int i = 0; i < kFM + kFN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, kFM * kFN, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // Stage s (parity P) of tile cur: step k runs while the fragments of step
  // k + 1 are read; before the last step every wave waits for its loads of
  // stage s + 1 (EXTRA younger operations may stay in flight) and the
  // barrier makes them visible and frees slot s % NS for stage s + NS, one
  // of the next tile's first where the tile ends.  No branch: a matrix
  // instruction would sink past one, and its operands spill.
  auto stage = [&](auto pc, auto extra, const Tile& cur, const Tile& nxt, int s) {
    constexpr int P = decltype(pc)::value;
    const int slot = NS == 2 ? P : s % NS, next = NS == 2 ? 1 - P : (s + 1) % NS;
    read_step(slot, 1);
    mma_step(pc, std::integral_constant<int, 0>{});
    phase_end();
    read_step(slot, 2);
    mma_step(pc, std::integral_constant<int, 1>{});
    phase_end();
    read_step(slot, 3);
    mma_step(pc, std::integral_constant<int, 2>{});
    phase_end();
    // loads issued after stage s + 1's: stages s + 2 .. s + NS - 1, the even ones with scales
    constexpr int kLater = [] {
      int n = decltype(extra)::value;
      for (int d = 2; d < NS; ++d) n += kL + ((P + d) % 2 == 0 ? kLS : 0);
      return n;
    }();
    wait_vmcnt_lgkm0<kLater>();
    raw_barrier();
    const bool over = s + NS >= ns;
    const Tile from = pick(over, nxt, cur);
    const int to = over ? s + NS - ns : s + NS;
    read_step(next, 0);
    mma_step(pc, std::integral_constant<int, 3>{});
    phase_end();
    if constexpr (P == 1) read_scales(((s + 1) / 2) % R::kScaleSlots);
    if constexpr ((P + NS) % 2 == 0) issue_scales(from, ((s + NS) / 2) % R::kScaleSlots, to / 2);
    issue_data(from, slot, to);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using Stores = std::integral_constant<int, kStores>;

  // The blocks of a walk finish their tiles together, and 256 CUs that store
  // 128 KB each at once wait for memory (a wave's stores retire before its
  // later loads).  Apart from each other by a quarter of a tile, the stores
  // of one group run under the products of the others.
  if constexpr (kWalk && kAct < 0) {
    for (int i = static_cast<int>(blockIdx.x * 4 / gridDim.x) * g.stagger; i > 0; --i) __builtin_amdgcn_s_sleep(32);
  }
  uint32_t t = blockIdx.x - kpart * count;
  Tile cur = tile_at(t);
  Tile none = cur;
  none.rows_m = none.rows_n = 0;
#pragma unroll
  for (int j = 0; j < kLS; ++j) none.s_bytes[j] = 0;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const Tile from = pick(s < ns, cur, none);
    const int at = s < ns ? s : 0;
    if (s % 2 == 0) issue_scales(from, s / 2, at / 2);
    issue_data(from, s, at);
  }
  wait_vmcnt_lgkm0<0>();
  raw_barrier();
  read_scales(0);
  read_step(0, 0);
  for (;;) {
    const Tile nxt = kWalk && t + gridDim.x < count ? tile_at(t + gridDim.x) : none;
#pragma unroll
    for (int i = 0; i < kFM; ++i)
#pragma unroll
      for (int j = 0; j < kFN; ++j) acc[i][j] = v16f{};
    // the stores of the tile before may still be in flight behind this tile's first two stages
    stage(I0{}, std::conditional_t<kWalk, Stores, I0>{}, cur, nxt, 0);
    stage(I1{}, I0{}, cur, nxt, 1);
    for (int s = 2; s < ns; s += 2) {
      stage(I0{}, I0{}, cur, nxt, s);
      stage(I1{}, I0{}, cur, nxt, s + 1);
    }

    // ---- epilogue: lane holds columns 32 j + 8 b + 4 grp + v of row 32 i + r32
    const int64_t mw = cur.m0 + wm * kWaveM, nw = cur.n0 + wn * kWaveN;
    auto bias_of = [&](int64_t n) { return g.bias && n < g.N ? bf16_to_f32(g.bias[n]) : 0.0f; };
    if constexpr (kAct >= 0) {
      const int64_t ldq = inter / 2;  // I % 32 == 0 (host)
      const int last = static_cast<int>(mx_tiles(inter)) * kMxTileBlocks, blocks = static_cast<int>(inter / kMxBlock);
      const int64_t cw = cur.n0 + wn * kHalf;  // the wave's first column
      if (cur.n0 + kTileN >= inter && wn == WN - 1) {  // the bytes of blocks past I (beyond the counted stores)
        for (int b = blocks; b < last; ++b)
#pragma unroll
          for (int i = 0; i < kFM; ++i) {
            const int64_t m = mw + 32 * i + r32;
            if (grp == 0 && m < g.M) g.s[((b >> 4) * g.M + m) * kMxTileBlocks + mx_scale_pos(b & 15)] = 0;
          }
      }
      const __amdgpu_buffer_rsrc_t rq = view(g.q + cur.m0 * ldq, cur.rows_m * ldq);
#pragma unroll
      for (int j = 0; j < kFN / 2; ++j) {
        const int64_t c = cw + 32 * j;
        const bool in = c < inter;  // whole blocks
        const int b = in ? static_cast<int>(c / kMxBlock) : 0;
        const __amdgpu_buffer_rsrc_t rs =
            view(g.s + ((b >> 4) * g.M + cur.m0) * kMxTileBlocks, in ? cur.rows_m * kMxTileBlocks : 0);
#pragma unroll
        for (int i = 0; i < kFM; ++i) {
          U16x8 lo, hi;  // columns 8 b + 4 grp + v, b = 0, 1 and b = 2, 3
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            float a[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float gate = static_cast<float>(static_cast<__bf16>(acc[i][j][2 * v + k]));
              const float up = static_cast<float>(static_cast<__bf16>(acc[i][j + kFN / 2][2 * v + k]));
              a[k] = mx_act_fn<kAct>(gate) * up;
            }
            const mx_bf16x2 p = {static_cast<__bf16>(a[0]), static_cast<__bf16>(a[1])};
            (v < 4 ? lo.w[v] : hi.w[v - 4]) = __builtin_bit_cast(uint32_t, p);
          }
          const uint32_t mine = mx_absmax8(lo), rest = mx_absmax8(hi), most = mine > rest ? mine : rest;
          const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
          const uint32_t byte = mx_scale_byte(both[0] > both[1] ? both[0] : both[1]);
          const float scale = mx_scale_value(byte == 255u ? 0u : byte);
          const uint32_t c01 = byte == 255u ? 0u : mx_codes8(lo, scale), c23 = byte == 255u ? 0u : mx_codes8(hi, scale);
          // lane l takes both lanes' codes of b = 0, 1, lane l + 32 those of b = 2, 3
          const auto x = __builtin_amdgcn_permlane32_swap(c01, c23, false, false);
          const int row = wm * kWaveM + 32 * i + r32;
          typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 codes = {(x[0] & 0xFFFFu) | (x[1] << 16), (x[0] >> 16) | (x[1] & 0xFFFF0000u)};
          __builtin_amdgcn_raw_buffer_store_b64(codes, rq, in ? static_cast<uint32_t>(row * ldq + c / 2 + 8 * grp) : 0x80000000u, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(byte), rs,
                                               grp == 0 ? row * kMxTileBlocks + mx_scale_pos(b & 15) : 0x80000000u, 0, 0);
          __builtin_amdgcn_sched_barrier(0);  // one fragment at a time: the next tile's operands are in registers already
        }
      }
    } else if constexpr (kSplit) {
      float* part = g.part + kpart * g.M * g.N;
#pragma unroll
      for (int i = 0; i < kFM; ++i) {
        const int64_t m = mw + 32 * i + r32;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < kFN; ++j)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int64_t n = nw + 32 * j + 8 * b + 4 * grp;  // N % 4 == 0 (host): 4 columns are all in or out
            if (n < g.N)
              *reinterpret_cast<v4f*>(part + m * g.N + n) =
                  v4f{acc[i][j][4 * b], acc[i][j][4 * b + 1], acc[i][j][4 * b + 2], acc[i][j][4 * b + 3]};
          }
      }
    } else if (g.store == 8) {
      // Lanes l and l + 32 swap halves: 8 adjacent columns of row 32 i + r32
      // each; then 16-lane groups swap between two such vectors: 16 rows of 64
      // contiguous bytes per 16-byte store.  Rows past M lie past the view.
      const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(
          scalar_ptr(g.out + cur.m0 * g.N), 0, static_cast<int>(cur.rows_m * g.N * 2), kBufferFlags);
#pragma unroll
      for (int j = 0; j < kFN; ++j) {
        float bias[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) bias[v] = 0.0f;
        if (g.bias) {
#pragma unroll
          for (int v = 0; v < 16; ++v) bias[v] = bias_of(nw + 32 * j + 8 * (v >> 2) + 4 * grp + (v & 3));
        }
#pragma unroll
        for (int i = 0; i < kFM; ++i) {
          uint32_t p[8];
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const mx_bf16x2 o = {static_cast<__bf16>(acc[i][j][2 * v] + bias[2 * v]),
                                 static_cast<__bf16>(acc[i][j][2 * v + 1] + bias[2 * v + 1])};
            p[v] = __builtin_bit_cast(uint32_t, o);
          }
          uint32_t o[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const auto x = __builtin_amdgcn_permlane32_swap(p[4 * h], p[4 * h + 2], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(p[4 * h + 1], p[4 * h + 3], false, false);
            o[h][0] = x[0];
            o[h][1] = y[0];
            o[h][2] = x[1];
            o[h][3] = y[1];
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const auto x = __builtin_amdgcn_permlane16_swap(o[0][k], o[1][k], false, false);
            o[0][k] = x[0];
            o[1][k] = x[1];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // rows 16 h + l % 16, lane groups 0 .. 3 on 8-column chunks 0, 2, 1, 3
            const int64_t n = nw + 32 * j + 8 * ((lane >> 4 & 1) * 2 + grp);
            const uint32_t off = n < g.N ? static_cast<uint32_t>(((wm * kWaveM + 32 * i + 16 * h + (lane & 15)) * g.N + n) * 2) : 0x80000000u;
            typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{o[h][0], o[h][1], o[h][2], o[h][3]}, ro, off, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      // four columns of a lane at a time, in one 8-byte store where rows allow
#pragma unroll
      for (int i = 0; i < kFM; ++i) {
        const int64_t m = mw + 32 * i + r32;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < kFN; ++j)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int64_t n = nw + 32 * j + 8 * b + 4 * grp;
            uint16_t o[4];
#pragma unroll
            for (int v = 0; v < 4; ++v)
              o[v] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(acc[i][j][4 * b + v] + bias_of(n + v)));
            uint16_t* at = g.out + m * g.N + n;
            if (g.store == 4) {
              if (n < g.N)
                *reinterpret_cast<uint2*>(at) = make_uint2(o[0] | static_cast<uint32_t>(o[1]) << 16, o[2] | static_cast<uint32_t>(o[3]) << 16);
            } else {
#pragma unroll
              for (int v = 0; v < 4; ++v)
                if (n + v < g.N) at[v] = o[v];
            }
          }
      }
      wait_vmcnt_lgkm0<0>();  // an uneven number of stores: none may hide a load of the next tile
    }
    t += gridDim.x;
    if (!kWalk || t >= count) break;
    cur = nxt;
  }
  wait_vmcnt_lgkm0<0>();  // no load into LDS outlives the block
#endif
}

// out = bf16(sum over p of part[p] + bias), added in the order of p; N % 4 == 0
__global__ __launch_bounds__(256) void mxfp4_split_sum_kernel(const float* __restrict__ part, int split, int64_t M, int64_t N,
                                                              const uint16_t* __restrict__ bias, uint16_t* __restrict__ out) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (e >= M * N) return;
  v4f s = *reinterpret_cast<const v4f*>(part + e);
#pragma unroll 4
  for (int p = 1; p < split; ++p) s += *reinterpret_cast<const v4f*>(part + p * M * N + e);
  if (bias) {
    const int64_t n = e % N;
#pragma unroll
    for (int v = 0; v < 4; ++v) s[v] += bf16_to_f32(bias[n + v]);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) out[e + v] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(s[v]));
#endif
}

}  // namespace
}  // namespace mw8
