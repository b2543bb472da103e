// MXFP4 products: y bf16 [M, N] = A W^T + bias of block-scaled 4-bit operands
// (format: mxfp4.h).  Up to 16 tokens, on many weight rows 32, stream the
// weights once (mxfp4_decode.h); more run on tile rings (mxfp4_ring.h), picked by
// a time model.
#include <algorithm>
#include <atomic>

#include "mxfp4_decode.h"

namespace mw8 {

int device_cus();
int quant_mxfp4_bf16(const void*, int64_t, int64_t, int64_t, uint8_t*, uint8_t*, hipStream_t);
int act_and_mul_quant_mxfp4_bf16(const void*, int64_t, int64_t, int, uint8_t*, uint8_t*, hipStream_t);

namespace {

// Raises the dynamic-LDS limit of kernel Kern once per device (the attribute
// is set on the current one).
template <auto Kern>
int mx_lds_limit(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error(kErrLaunch, "hipGetDevice: %s", hipGetErrorString(e));
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t{1} << dev : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit) != 0) return kOk;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return set_error(kErrLaunch, "hipFuncSetAttribute(%d bytes of LDS): %s", bytes, hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_acq_rel);
  return kOk;
}

inline bool aligned_to(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kLdsBytes = 163840;

// ------------------------------------------------------------------- rings
// Tilings and what the time model knows of them (MI355X, fitted to graph-timed
// runs of 130 random shapes from 17 to 8192 rows): us = start + (rounds - 1)
// round + max(latency stages rounds, rate stages tiles per CU), at least
// start + the operands and the output at bw TB/s.  On the shapes it was
// fitted to the pick is 0.5% off the fastest configuration on average and 13% at
// most (78 x 51200 x 5120).
struct MxRingCfg {
  int bm, bn, per_cu;
  float start, round, latency, rate, bw;
};
constexpr MxRingCfg kMxRings[] = {
    {256, 256, 1, 5.19f, 6.50f, 1.559f, 1.608f, 3.40f},  // 0: a block per CU walks its tiles
    {256, 192, 1, 4.44f, 4.27f, 1.308f, 0.914f, 3.52f},  // 1: likewise
    {128, 128, 2, 3.79f, 2.20f, 0.695f, 0.588f, 3.64f},  // 2: likewise, two blocks per CU
    {128, 128, 1, 4.23f, 3.95f, 0.573f, 0.397f, 4.32f},  // 3: four stages in flight
    {64, 64, 2, 3.38f, 1.55f, 0.271f, 0.243f, 5.11f},    // 4: likewise; the one that splits K
};
constexpr int kNumMxRings = sizeof(kMxRings) / sizeof(kMxRings[0]);
constexpr int kMxSplitCfg = 4, kMxMaxSplit = 16, kMxDecodeRows = 16;

struct MxPlan {
  int cfg, split;  // cfg < 0: a decode kernel
};

// The decode kernel whose blocks keep the tokens in LDS: waves per block (0: the
// others are faster) and ring slots per wave.  It pays from 96 weight rows per
// CU on, for 8 tokens and more, up to 12 tiles of them (MI355X, us, this / the
// other: 16 x 24576 x 5120 13.8 / 14.7, 32 rows 14.5 / 18.3; 8 x 34816 x 5120 18.5 /
// 19.3; 16 x 40000 x 1024 7.3 / 10.3; but 32 x 16384 x 2048 6.8 / 6.5, 5 x 58208 x
// 1568 15.4 / 13.7, 16 x 32768 x 8192 31 / 27; 14 random shapes within the rule 0.66
// to 1.04 of the other's time).  As many waves as give each
// chunks of 16 rows, with two slots where the LDS holds them (16 x 24576 x 5120,
// 6 waves: two slots 13.8, one 14.3; 8 waves, 12 rows each: 13.9).
struct MxSharedPlan {
  int waves, depth;
};
constexpr int kMxSharedRows = 32;
MxSharedPlan mx_shared_plan(int64_t M, int64_t N, int64_t K) {
  const int64_t cus = device_cus(), tiles = mx_tiles(K);
  // (chunks are counted in 32 bits)
  if (M < 8 || M > kMxSharedRows || N < 96 * cus || N >= (1ll << 26) || tiles > 12) return {0, 0};
  const int64_t rows = (N + cus - 1) / cus;
  const int64_t room = (kLdsBytes - tiles * (M > 16 ? 2 : 1) * (kMxSlot + 256)) / kMxSlot;
  const int64_t most = std::min<int64_t>(room, 16), chunks = (rows + 16 * most - 1) / (16 * most);
  const int64_t waves = (rows + 16 * chunks - 1) / (16 * chunks);
  return {static_cast<int>(waves), 2 * waves <= room ? 2 : 1};
}

thread_local int g_mx_cfg = -1, g_mx_split = 0;  // override of the calling thread (-1: automatic)

double mx_ring_us(int c, int64_t M, int64_t N, int64_t K, int split) {
  const MxRingCfg& r = kMxRings[c];
  const int64_t cus = device_cus(), tiles = ((M + r.bm - 1) / r.bm) * ((N + r.bn - 1) / r.bn) * split;
  const double stages = 2.0 * ((mx_tiles(K) + split - 1) / split);
  const double rounds = static_cast<double>((tiles + cus * r.per_cu - 1) / (cus * r.per_cu)),
               per_cu = static_cast<double>((tiles + cus - 1) / cus);
  double us = r.start + (rounds - 1) * r.round + std::max(r.latency * stages * rounds, r.rate * stages * per_cu);
  const double bytes = static_cast<double>(N) * K * (17.0 / 32) + 2.0 * M * N;
  us = std::max(us, r.start + bytes / (r.bw * 1e6));
  // the sums' way through memory and the second launch
  if (split > 1) us += 2.1 + 8.0 * split * M * N / 3.9e6;
  return us;
}

// The ring that the time model finds fastest, and its time.
MxPlan mx_fastest_ring(int64_t M, int64_t N, int64_t K, bool may_split, double& us) {
  const int64_t tiles = mx_tiles(K);
  MxPlan best{0, 1};
  us = 1e30;
  for (int c = 0; c < kNumMxRings; ++c) {
    const int most = may_split && c == kMxSplitCfg ? static_cast<int>(std::min<int64_t>(kMxMaxSplit, tiles)) : 1;
    for (int s = 1; s <= most; ++s) {
      const double t = mx_ring_us(c, M, N, K, s);
      if (t < us) {
        us = t;
        best = {c, s};
      }
    }
  }
  return best;
}

MxPlan mx_plan(int64_t M, int64_t N, int64_t K, bool may_split) {
  may_split = may_split && N % 4 == 0;
  if (g_mx_cfg >= 0) {
    const bool split = may_split && g_mx_cfg == kMxSplitCfg && g_mx_split > 1 && g_mx_split <= mx_tiles(K);
    return {g_mx_cfg, split ? g_mx_split : 1};
  }
  if (M <= kMxDecodeRows || mx_shared_plan(M, N, K).waves > 0) return {-1, 1};
  double us;
  return mx_fastest_ring(M, N, K, may_split, us);
}

template <int BM, int BN, int WM, int WN, int NS, bool kSplit = false, int kAct = -1>
int launch_ring(MxArgs g, hipStream_t st) {
  using R = MxRing<BM, BN, WM, WN, NS>;
  constexpr auto kern = mxfp4_ring_kernel<BM, BN, WM, WN, NS, kSplit, kAct>;
  constexpr int kThreads = 64 * R::kWaves;
  const int64_t tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN /* kAct: ceil(I / (BN / 2)) */,
                slots = device_cus() * (kLdsBytes / R::kLds);
  MW8_REQUIRE(tm < (1ll << 29) && tn < (1ll << 29) && tm * tn * g.split < (1ll << 31), kErrShape,
              "gemm_mxfp4: M=%lld x N=%lld too large", (long long)g.M, (long long)g.N);
  g.raster = MxRaster::of(tm, tn);
  const int64_t all = tm * tn * g.split, blocks = NS == 2 ? std::min(all, slots) : all;
  MW8_REQUIRE(blocks * kThreads < (1ll << 32), kErrShape, "gemm_mxfp4: M=%lld x N=%lld too large", (long long)g.M,
              (long long)g.N);
  // From eight rounds and K = 4096 on the last group's late start costs less
  // than the stores' bursts (MI355X, us, together -> staggered: 8192 x 34816 x
  // 5120 748 -> 716, 4096 rows 391 -> 369, 8192 x 51200 x 5120 1139 -> 1125; but 2080
  // x 51200 x 5120, 7 rounds, 310 -> 318, and 8192 x 16384 x 2048 159 -> 171).
  if (BM == 256 && BN == 256 && tm * tn >= 8 * blocks && g.tiles >= 8) g.stagger = g.tiles * 4 / 5;
  if (const int rc = mx_lds_limit<kern>(R::kLds)) return rc;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), R::kLds, st, g);
  return check_launch("gemm_mxfp4");
}

int run_ring(const MxArgs& g, int cfg, hipStream_t st) {
  switch (cfg) {
    case 0: return launch_ring<256, 256, 4, 2, 2>(g, st);
    case 1: return launch_ring<256, 192, 4, 2, 2>(g, st);
    case 2: return launch_ring<128, 128, 2, 2, 2>(g, st);
    case 3: return launch_ring<128, 128, 2, 2, 4>(g, st);
    default: break;
  }
  if (g.split == 1) return launch_ring<64, 64, 2, 2, 4>(g, st);
  if (const int rc = launch_ring<64, 64, 2, 2, 4, true>(g, st)) return rc;
  const int64_t blocks = (g.M * g.N / 4 + 255) / 256;
  MW8_REQUIRE(blocks < (1ll << 24), kErrShape, "gemm_mxfp4: M=%lld x N=%lld too large to split", (long long)g.M,
              (long long)g.N);
  hipLaunchKernelGGL(mxfp4_split_sum_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, g.part, g.split, g.M,
                     g.N, g.bias, g.out);
  return check_launch("gemm_mxfp4");
}

// ------------------------------------------------------------------ decode
// 16-row groups per block and 512-element tiles per wave.  Two row groups
// share the tokens' fragments and leave N <= 32 x CUs one block per CU (MI355X,
// us, one -> two groups: 16 x 16384 x 5120 12.1 -> 10.8, 16 x 5120 x 17408
// 15.5 -> 12.8); few tokens and more rows than that are faster in single
// groups (1 x 34816 x 5120 18.6 -> 17.6, 8 tokens 19.7 -> 19.2).  Four tiles
// per wave, two where single groups have enough waves (1 x 34816 x 5120 18.3
// -> 17.6), more where the waves' rings would not fit the LDS.
struct MxDecodePlan {
  int groups, per_wave, waves;
};
MxDecodePlan mx_decode_plan(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = mx_tiles(K);
  const int groups = M > 8 || N <= 32 * static_cast<int64_t>(device_cus()) ? 2 : 1;
  int64_t per = tiles >= 8 ? (groups == 1 ? 2 : 4) : tiles >= 4 ? 2 : 1;
  const int64_t most = groups == 2 ? 9 : 16, need = (tiles + most - 1) / most;
  if (per < need) per = need;
  return {groups, static_cast<int>(per), static_cast<int>((tiles + per - 1) / per)};
}

constexpr int kMxDepth = 2;  // tiles in flight per wave: 3 or 4 were 5-15% slower (fewer blocks fit the LDS)

int mx_decode_lds(const MxDecodePlan& p, int64_t M, int64_t K, bool xq) {
  const int ring = p.waves * kMxDepth * p.groups * kMxSlot, sums = p.waves * 16 * (16 * p.groups + 1) * 4;
  return std::max(ring, sums) + (xq ? static_cast<int>(mx_tiles(K) * M * 272) : 0);
}

template <int RG, bool kXQ>
int launch_decode(const MxDecodeArgs& d, const MxDecodePlan& p, hipStream_t st) {
  constexpr auto kern = mxfp4_decode_kernel<RG, kMxDepth, kXQ>;
  const int lds = mx_decode_lds(p, d.g.M, d.K, kXQ);
  if (const int rc = mx_lds_limit<kern>(kLdsBytes)) return rc;
  const int64_t cus = device_cus(), blocks = cus * ((d.g.N + cus * 16 * RG - 1) / (cus * 16 * RG));
  MW8_REQUIRE(blocks * 64 * p.waves < (1ll << 32), kErrShape, "gemm_mxfp4: N=%lld x K=%lld too large", (long long)d.g.N,
              (long long)d.K);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(64 * p.waves), lds, st, d);
  return check_launch("gemm_mxfp4");
}

template <int TG, int D>
int launch_decode_shared(const MxArgs& g, int waves, hipStream_t st) {
  constexpr auto kern = mxfp4_decode_shared_kernel<TG, D>;
  if (const int rc = mx_lds_limit<kern>(kLdsBytes)) return rc;
  const int lds = g.tiles * TG * (kMxSlot + 256) + waves * D * kMxSlot;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(device_cus())), dim3(64 * waves), lds, st, g);
  return check_launch("gemm_mxfp4");
}

MxArgs mx_args(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, const void* bias, void* y,
               int64_t M, int64_t N, int64_t K) {
  // (16-byte stores go through a 32-bit view of a tile's output rows)
  const int store = N % 8 == 0 && aligned_to(y, 16) && N < (1ll << 22) ? 8 : N % 4 == 0 && aligned_to(y, 8) ? 4 : 1;
  return {A, sa, W, sw, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(y), M, N,
          static_cast<int>(mx_blocks(K)), static_cast<int>(mx_tiles(K)), store, {}, nullptr, 1, 0, nullptr, nullptr};
}

}  // namespace

void set_mxfp4_tuning(int cfg, int split) {
  g_mx_cfg = cfg >= 0 && cfg < kNumMxRings ? cfg : -1;
  g_mx_split = split;
}
int mxfp4_tuning_count() { return kNumMxRings; }

size_t gemm_mxfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const MxPlan p = mx_plan(M, N, K, true);
  return p.split > 1 ? static_cast<size_t>(p.split) * M * N * 4 : 0;
}

int gemm_mxfp4_bf16(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, const void* bias, void* y,
                    int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes, hipStream_t st) {
  MW8_REQUIRE(A && sa && W && sw && y, kErrArg, "gemm_mxfp4: null pointer");
  MW8_REQUIRE(M >= 0 && N > 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K <= (1ll << 20), kErrShape,
              "gemm_mxfp4: bad sizes M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  MW8_REQUIRE(aligned_to(A, 16) && aligned_to(W, 16) && aligned_to(sa, 16) && aligned_to(sw, 16) && aligned_to(y, 2) &&
                  aligned_to(bias, 2) && aligned_to(ws, 16),
              kErrAlign, "gemm_mxfp4: A, sa, W, sw and the workspace need 16-byte, y and bias 2-byte alignment");
  if (M == 0) return kOk;
  MW8_REQUIRE(!any_meet({one_row(y, M * N * 2)}, {mx_codes_mem(A, M, K), mx_scales_mem(sa, M, K), mx_codes_mem(W, N, K),
                                                 mx_scales_mem(sw, N, K), one_row(bias, N * 2)}),
              kErrArg, "gemm_mxfp4: y must not overlap an input");
  MxArgs g = mx_args(A, sa, W, sw, bias, y, M, N, K);
  const MxPlan p = mx_plan(M, N, K, ws != nullptr);
  if (p.cfg < 0) {
    if (const MxSharedPlan sp = mx_shared_plan(M, N, K); sp.waves > 0) {
      if (M > 16) return sp.depth == 2 ? launch_decode_shared<2, 2>(g, sp.waves, st) : launch_decode_shared<2, 1>(g, sp.waves, st);
      return sp.depth == 2 ? launch_decode_shared<1, 2>(g, sp.waves, st) : launch_decode_shared<1, 1>(g, sp.waves, st);
    }
    const MxDecodePlan dp = mx_decode_plan(M, N, K);
    const MxDecodeArgs d{g, nullptr, 0, K, dp.per_wave};
    return dp.groups == 2 ? launch_decode<2, false>(d, dp, st) : launch_decode<1, false>(d, dp, st);
  }
  if (p.split > 1) {
    const size_t need = static_cast<size_t>(p.split) * M * N * 4;
    MW8_REQUIRE(ws_bytes >= need, kErrWorkspace, "gemm_mxfp4: the workspace holds %zu of %zu bytes", ws_bytes, need);
    MW8_REQUIRE(!any_meet({one_row(ws, static_cast<int64_t>(need))},
                          {one_row(y, M * N * 2), mx_codes_mem(A, M, K), mx_scales_mem(sa, M, K), mx_codes_mem(W, N, K),
                           mx_scales_mem(sw, N, K), one_row(bias, N * 2)}),
                kErrArg, "gemm_mxfp4: the workspace must not overlap y or an input");
    g.part = static_cast<float*>(ws);
    g.split = p.split;
  }
  return run_ring(g, p.cfg, st);
}

// Whether gemm_act_mxfp4 takes (M, I, K): whole blocks of activation columns,
// the weight and 256 rows of codes within 32-bit views.
int gemm_act_mxfp4_supported(int64_t M, int64_t I, int64_t K) {
  return M > 0 && I > 0 && K > 0 && K <= (1ll << 20) && I % kMxBlock == 0 && I < (1ll << 24) &&
         2 * I * mx_blocks(K) * 16 < (1ll << 31) && M < (1ll << 31);
}

// Whether it is the faster way to the quantized activation, against the plain
// product and act_and_mul_quant_mxfp4.  Fused: 6 us, and per round of 256-row x
// 128-column tiles 3 us + 1.6 us a stage (MI355X, us, fused / two launches: 200 x
// 25600 x 5120 49 / 69, 2080 rows 294 / 369; 333 x 17408 75 / 63, 2080 rows 193 /
// 236; 1024 x 6400 39 / 49; K = 2048: 1024 x 768 18 / 13, 8192 rows 22 / 31).  Never
// where the product would run on a decode kernel (17 rows: 32768 x 5120 45 / 32, 16384 x
// 5120 35 / 19, 32768 x 512 11.7 / 10.2).
int gemm_act_mxfp4_preferred(int64_t M, int64_t I, int64_t K) {
  if (M <= kMxDecodeRows || !gemm_act_mxfp4_supported(M, I, K) || mx_shared_plan(M, 2 * I, K).waves > 0) return 0;
  const int64_t cus = device_cus(), tiles = ((M + 255) / 256) * ((I + 127) / 128);
  const double rounds = static_cast<double>((tiles + cus - 1) / cus);
  const double fused = 6.0 + rounds * (3.0 + 1.6 * 2 * mx_tiles(K));
  double us;
  mx_fastest_ring(M, 2 * I, K, true, us);
  return fused < us + 2.5 + 4.53 * M * I / 5.5e6;
}

int gemm_act_mxfp4(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int act, uint8_t* q, uint8_t* s,
                   int64_t M, int64_t I, int64_t K, hipStream_t st) {
  MW8_REQUIRE(A && sa && W && sw && q && s, kErrArg, "gemm_act_mxfp4: null pointer");
  MW8_REQUIRE(act == 0 || act == 1, kErrArg, "gemm_act_mxfp4: act must be 0 (silu) or 1 (gelu)");
  MW8_REQUIRE(M >= 0, kErrShape, "gemm_act_mxfp4: bad size M=%lld", (long long)M);
  if (M == 0) return kOk;
  MW8_REQUIRE(gemm_act_mxfp4_supported(M, I, K), kErrShape, "gemm_act_mxfp4: M=%lld I=%lld K=%lld not supported", (long long)M,
              (long long)I, (long long)K);
  MW8_REQUIRE(aligned_to(A, 16) && aligned_to(W, 16) && aligned_to(sa, 16) && aligned_to(sw, 16) && aligned_to(q, 8), kErrAlign,
              "gemm_act_mxfp4: A, sa, W and sw need 16-byte and q 8-byte alignment");
  MW8_REQUIRE(!any_meet({mx_codes_mem(q, M, I), mx_scales_mem(s, M, I)},
                        {mx_codes_mem(A, M, K), mx_scales_mem(sa, M, K), mx_codes_mem(W, 2 * I, K), mx_scales_mem(sw, 2 * I, K)}),
              kErrArg, "gemm_act_mxfp4: q and s must not overlap each other or an input");
  MxArgs g = mx_args(A, sa, W, sw, nullptr, nullptr, M, 2 * I, K);
  g.q = q;
  g.s = s;
  return act == 0 ? launch_ring<256, 256, 4, 2, 2, false, 0>(g, st) : launch_ring<256, 256, 4, 2, 2, false, 1>(g, st);
}

// Whether linear_bf16_mxfp4 takes (M, N, K): few enough rows for each wave's
// passes (half of them in single row groups, where a CU runs several blocks:
// 4 x 5120 -> 34816 21.6 us, in two launches 20.4, 2 rows 19.6 and 20.2), their
// codes beside the weight ring in the LDS, K in whole 16-byte vectors.
int linear_bf16_mxfp4_supported(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || M > kMxPasses || N < 1 || N >= (1ll << 31) || K < 8 || K % 8 != 0 || K > (1ll << 20)) return 0;
  const MxDecodePlan p = mx_decode_plan(M, N, K);
  return g_mx_cfg < 0 && M * p.per_wave <= (p.groups == 2 ? kMxPasses : kMxPasses / 2) &&
         mx_decode_lds(p, M, K, true) <= kLdsBytes;
}

// Rows that it can read: whole 16-byte vectors within a 32-bit view.
static bool linear_takes(const void* x, int64_t ldx, int64_t M) {
  return aligned_to(x, 16) && (M == 1 || (ldx % 8 == 0 && ldx < (1ll << 26)));
}

int linear_bf16_mxfp4(const void* x, int64_t ldx, const uint8_t* W, const uint8_t* sw, const void* bias, void* y, int64_t M,
                      int64_t N, int64_t K, hipStream_t st) {
  MW8_REQUIRE(x && W && sw && y, kErrArg, "linear_mxfp4: null pointer");
  MW8_REQUIRE(M >= 0 && N > 0 && K > 0 && ldx >= K && (M == 1 || ldx < (1ll << 26)), kErrShape,
              "linear_mxfp4: bad sizes M=%lld N=%lld K=%lld ldx=%lld", (long long)M, (long long)N, (long long)K, (long long)ldx);
  if (M == 0) return kOk;
  MW8_REQUIRE(linear_bf16_mxfp4_supported(M, N, K), kErrShape, "linear_mxfp4: M=%lld N=%lld K=%lld not supported",
              (long long)M, (long long)N, (long long)K);
  MW8_REQUIRE(aligned_to(x, 16) && (M == 1 || ldx % 8 == 0) && aligned_to(W, 16) && aligned_to(sw, 16) && aligned_to(y, 2) &&
                  aligned_to(bias, 2),
              kErrAlign, "linear_mxfp4: x, its rows, W and sw need 16-byte, y and bias 2-byte alignment");
  MW8_REQUIRE(!any_meet({one_row(y, M * N * 2)}, {RowSet{x, 2 * K, M, 2 * ldx, 1, 0}, mx_codes_mem(W, N, K),
                                                 mx_scales_mem(sw, N, K), one_row(bias, N * 2)}),
              kErrArg, "linear_mxfp4: y must not overlap an input");
  const MxDecodePlan dp = mx_decode_plan(M, N, K);
  const MxDecodeArgs d{mx_args(nullptr, nullptr, W, sw, bias, y, M, N, K), static_cast<const uint16_t*>(x), M == 1 ? K : ldx, K,
                       dp.per_wave};
  return dp.groups == 2 ? launch_decode<2, true>(d, dp, st) : launch_decode<1, true>(d, dp, st);
}

namespace {

// The gated MLP's buffers between its launches, from the start of the workspace
// (bytes; 256-byte aligned).
struct MxMlpPlan {
  bool act_in_product;
  size_t xq, xs, gate_up, aq, as, part, part_bytes, total;
};
MxMlpPlan mx_mlp_plan(bool quantized, int64_t M, int64_t H, int64_t I, int64_t N) {
  MxMlpPlan p{};
  p.act_in_product = gemm_act_mxfp4_preferred(M, I, H) != 0;
  auto take = [&](size_t bytes) {
    const size_t at = p.total;
    p.total += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t m = static_cast<size_t>(M);
  p.xq = take(quantized ? 0 : m * mx_blocks(H) * 16);
  p.xs = take(quantized ? 0 : m * mx_tiles(H) * kMxTileBlocks);
  p.gate_up = take(p.act_in_product ? 0 : m * I * 4);
  p.aq = take(m * mx_blocks(I) * 16);
  p.as = take(m * mx_tiles(I) * kMxTileBlocks);
  p.part_bytes = std::max(p.act_in_product ? 0 : gemm_mxfp4_workspace_bytes(M, 2 * I, H), gemm_mxfp4_workspace_bytes(M, N, I));
  p.part = take(p.part_bytes);
  return p;
}

bool mx_mlp_sizes(int64_t M, int64_t H, int64_t I, int64_t N) {
  return M >= 0 && H > 0 && I > 0 && N > 0 && M < (1ll << 31) && H <= (1ll << 20) && I <= (1ll << 20) && N < (1ll << 31);
}

}  // namespace

size_t gated_mlp_mxfp4_workspace_bytes(int quantized, int64_t M, int64_t H, int64_t I, int64_t N) {
  return M > 0 && mx_mlp_sizes(M, H, I, N) ? mx_mlp_plan(quantized != 0, M, H, I, N).total : 0;
}

int gated_mlp_mxfp4(const void* x, int64_t ldx, const uint8_t* q, const uint8_t* s, const uint8_t* Wg, const uint8_t* sg,
                    const uint8_t* Wd, const uint8_t* sd, int act, void* y, int64_t M, int64_t H, int64_t I, int64_t N,
                    void* ws, size_t ws_bytes, hipStream_t st) {
  MW8_REQUIRE((x || (q && s)) && Wg && sg && Wd && sd && y, kErrArg, "gated_mlp_mxfp4: null pointer");
  MW8_REQUIRE(act == 0 || act == 1, kErrArg, "gated_mlp_mxfp4: act must be 0 (silu) or 1 (gelu)");
  MW8_REQUIRE(mx_mlp_sizes(M, H, I, N) && (!x || ldx >= H), kErrShape, "gated_mlp_mxfp4: bad sizes M=%lld H=%lld I=%lld N=%lld",
              (long long)M, (long long)H, (long long)I, (long long)N);
  if (M == 0) return kOk;
  const MxMlpPlan p = mx_mlp_plan(!x, M, H, I, N);
  MW8_REQUIRE(ws && ws_bytes >= p.total, kErrWorkspace, "gated_mlp_mxfp4: the workspace holds %zu of %zu bytes", ws ? ws_bytes : 0,
              p.total);
  MW8_REQUIRE(aligned_to(ws, 16), kErrAlign, "gated_mlp_mxfp4: the workspace needs 16-byte alignment");
  const RowSet none = one_row(nullptr, 0);
  MW8_REQUIRE(!any_meet({one_row(y, M * N * 2), one_row(ws, static_cast<int64_t>(p.total))},
                        {x ? RowSet{x, 2 * H, M, 2 * ldx, 1, 0} : none, x ? none : mx_codes_mem(q, M, H),
                         x ? none : mx_scales_mem(s, M, H), mx_codes_mem(Wg, 2 * I, H), mx_scales_mem(sg, 2 * I, H),
                         mx_codes_mem(Wd, N, I), mx_scales_mem(sd, N, I)}),
              kErrArg, "gated_mlp_mxfp4: y and the workspace must not overlap each other or an input");
  auto* b = static_cast<uint8_t*>(ws);
  void* part = p.part_bytes > 0 ? b + p.part : nullptr;
  void* gu = b + p.gate_up;
  const bool one = x && linear_takes(x, ldx, M) && linear_bf16_mxfp4_supported(M, 2 * I, H);
  if (x && !one) {
    if (const int rc = quant_mxfp4_bf16(x, M, H, ldx, b + p.xq, b + p.xs, st)) return rc;
    q = b + p.xq;
    s = b + p.xs;
  }
  if (p.act_in_product) {
    if (const int rc = gemm_act_mxfp4(q, s, Wg, sg, act, b + p.aq, b + p.as, M, I, H, st)) return rc;
  } else {
    if (const int rc = one ? linear_bf16_mxfp4(x, ldx, Wg, sg, nullptr, gu, M, 2 * I, H, st)
                           : gemm_mxfp4_bf16(q, s, Wg, sg, nullptr, gu, M, 2 * I, H, part, p.part_bytes, st))
      return rc;
    if (const int rc = act_and_mul_quant_mxfp4_bf16(gu, M, 2 * I, act, b + p.aq, b + p.as, st)) return rc;
  }
  return gemm_mxfp4_bf16(b + p.aq, b + p.as, Wd, sd, nullptr, y, M, N, I, part, p.part_bytes, st);
}

}  // namespace mw8
