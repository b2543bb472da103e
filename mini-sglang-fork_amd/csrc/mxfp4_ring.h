// MXFP4 tile ring: BM x BN output tiles whose operands stream through LDS.
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

template <int BM, int BN, int WM, int WN, int NS, bool kSplit>
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
  constexpr int kStores = kFM * kFN * 2;                 // 16-byte store instructions per wave and tile
  constexpr bool kWalk = NS == 2;                        // a block walks tiles blockIdx, blockIdx + gridDim, ...
  static_assert(kLA * 8 * kWaves == BM && kLB * 8 * kWaves == BN && BM % 64 == 0 && BN % 64 == 0, "DMA split");
  static_assert(!kSplit || !kWalk, "a split block owns one tile");
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
  struct Tile {
    int64_t m0, n0;
    const uint8_t *a, *w, *sa, *sw;
    int rows_m, rows_n;  // 0: no tile, every load reads zeros
  };
  auto tile_at = [&](uint32_t t) {
    Tile o;
    uint32_t pm, pn;
    const bool live = t < count;
    g.raster.tile(live ? t : 0, pm, pn);
    o.m0 = static_cast<int64_t>(pm) * BM;
    o.n0 = static_cast<int64_t>(pn) * BN;
    o.a = g.A + o.m0 * ld;
    o.w = g.W + o.n0 * ld;
    o.sa = g.sa + o.m0 * 16;
    o.sw = g.sw + o.n0 * 16;
    o.rows_m = live ? static_cast<int>(g.M - o.m0 < BM ? g.M - o.m0 : BM) : 0;
    o.rows_n = live ? static_cast<int>(g.N - o.n0 < BN ? g.N - o.n0 : BN) : 0;
    return o;
  };
  // field by field (a choice between two references would put both in memory)
  auto pick = [](bool c, const Tile& x, const Tile& y) {
    return Tile{c ? x.m0 : y.m0, c ? x.n0 : y.n0,         c ? x.a : y.a,          c ? x.w : y.w,
                c ? x.sa : y.sa, c ? x.sw : y.sw, c ? x.rows_m : y.rows_m, c ? x.rows_n : y.rows_n};
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
    w_off[j] = static_cast<uint32_t>(row * ld + 16 * ((unit & 7) ^ swz_f<128>(row)));
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
  // scales of the tile's 512 elements number p: instruction u fills rows
  // 64 u .. 64 u + 63 of the slot (the tile's A rows, then its W rows)
  auto issue_scales = [&](const Tile& o, int slot, int p) {
    const int64_t t = kt0 + p;
    unsigned char* base = lds + NS * R::kStage + slot * R::kScale;
#pragma unroll
    for (int j = 0; j < kLS; ++j) {
      const int u = j * kWaves + wave < kSUnits ? j * kWaves + wave : kSUnits - 1;
      const bool is_a = u < BM / 64;
      const int row = (is_a ? u : u - BM / 64) * 64;
      const int rows = is_a ? o.rows_m : o.rows_n;
      const __amdgpu_buffer_rsrc_t rs =
          view(is_a ? o.sa + t * g.M * 16 : o.sw + t * g.N * 16, rows * 16);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(base + u * 1024), 16, row * 16 + lane * 16, 0, 0, 0);
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

  uint32_t t = blockIdx.x - kpart * count;
  Tile cur = tile_at(t);
  Tile none = cur;
  none.rows_m = none.rows_n = 0;
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
    if constexpr (kSplit) {
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
      // lanes l and l + 32 swap halves: 8 adjacent columns of row 32 i + r32
      // each, one 16-byte store; rows past M lie past the view
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
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const auto x = __builtin_amdgcn_permlane32_swap(p[4 * h], p[4 * h + 2], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(p[4 * h + 1], p[4 * h + 3], false, false);
            const int64_t n = nw + 32 * j + 16 * h + 8 * grp;
            const uint32_t off = n < g.N ? static_cast<uint32_t>(((wm * kWaveM + 32 * i + r32) * g.N + n) * 2) : 0x80000000u;
            typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], y[0], x[1], y[1]}, ro, off, 0, 0);
          }
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
