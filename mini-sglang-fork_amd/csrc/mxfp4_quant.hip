// MXFP4 quantizer, gated activation + quantizer, and dequantizer (gfx950).
//
// A block of 32 needs its own 32 values only, so there is no row reduction:
// one wave takes U rows of one 512-element tile (lane l holds elements
// 8 l .. 8 l + 7, a quad of lanes holds a block), reads 1 KB and writes 256
// code bytes per row, and the tile's 16 scale bytes.  Everything is read and
// written once; the bound is HBM (MI355X, 8192 x 17408: quantizer 58-62 us, 5.9-6.2
// TB/s; dequantizer 60-70 us, 5.2-6.0; silu + quantizer 105-112 us, 5.8-6.1; gelu +
// quantizer 124-140 us, bound by the activation's instructions).
#include "mxfp4.h"

namespace mw8 {

namespace {

constexpr int kMxThreads = 256;
constexpr int kMxWaves = kMxThreads / 64;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// 8 bf16 elements k .. k + 7 of a row of K (zeros past K).  VEC: the row is
// 16-byte aligned and K % 8 == 0, so the 8 are all in or all out.
template <bool VEC>
__device__ __forceinline__ U16x8 mx_load8(const uint16_t* row, int64_t k, int64_t K) {
  U16x8 v;
  if constexpr (VEC) {
    u32x4 w = {0, 0, 0, 0};
    if (k < K) w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + k));
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = w[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = k + 2 * j < K ? row[k + 2 * j] : 0u, hi = k + 2 * j + 1 < K ? row[k + 2 * j + 1] : 0u;
      v.w[j] = lo | (hi << 16);
    }
  }
  return v;
}

// ACT < 0: x [M, K] at row stride ldx.  ACT >= 0: x [M, 2K] (gate | up),
// quantized is bf16(act(gate) * up).
template <int U, bool VEC, int ACT>
__global__ __launch_bounds__(kMxThreads) void quant_mxfp4_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t M,
                                                                 int64_t K, uint8_t* __restrict__ q,
                                                                 uint8_t* __restrict__ s) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63;
  const uint32_t tiles = static_cast<uint32_t>(mx_tiles(K));
  const uint32_t item = blockIdx.x * kMxWaves + (threadIdx.x >> 6);
  const uint32_t kt = item % tiles;
  const int64_t r0 = static_cast<int64_t>(item / tiles) * U;
  const int64_t ldq = mx_blocks(K) * 16;
  const int64_t k = static_cast<int64_t>(kt) * kMxTile + 8 * lane;
  U16x8 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u < M ? r0 + u : (M - 1);
    v[u] = mx_load8<VEC>(x + r * ldx, k, K);
    if constexpr (ACT >= 0) {
      const U16x8 up = mx_load8<VEC>(x + r * ldx + K, k, K);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const mx_bf16x2 a = {static_cast<__bf16>(mx_act_fn<ACT>(bf16_lo(v[u].w[j])) * bf16_lo(up.w[j])),
                             static_cast<__bf16>(mx_act_fn<ACT>(bf16_hi(v[u].w[j])) * bf16_hi(up.w[j]))};
        v[u].w[j] = __builtin_bit_cast(uint32_t, a);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t byte;
    const uint32_t codes = mx_quant_quad(v[u], byte);
    if (r0 + u >= M) break;  // wave-uniform
    if (k / 2 < ldq) __builtin_nontemporal_store(codes, reinterpret_cast<uint32_t*>(q + (r0 + u) * ldq + k / 2));
    if ((lane & 3) == 0) s[(static_cast<int64_t>(kt) * M + r0 + u) * 16 + mx_scale_pos(lane >> 2)] = static_cast<uint8_t>(byte);
  }
#endif
}

// y[m, k] = code value * 2^e as bf16 (exact down to bf16's subnormals)
template <bool VEC>
__global__ __launch_bounds__(kMxThreads) void dequant_mxfp4_kernel(const uint8_t* __restrict__ q,
                                                                   const uint8_t* __restrict__ s, int64_t M, int64_t K,
                                                                   uint16_t* __restrict__ y) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63;
  const uint32_t tiles = static_cast<uint32_t>(mx_tiles(K));
  const uint32_t item = blockIdx.x * kMxWaves + (threadIdx.x >> 6);
  const uint32_t kt = item % tiles;
  const int64_t r = item / tiles;
  const int64_t ldq = mx_blocks(K) * 16;
  const int64_t k = static_cast<int64_t>(kt) * kMxTile + 8 * lane;
  if (r >= M || k >= K) return;
  const uint32_t codes = *reinterpret_cast<const uint32_t*>(q + r * ldq + k / 2);
  const uint32_t byte = s[(static_cast<int64_t>(kt) * M + r) * 16 + mx_scale_pos(lane >> 2)];
  const float scale = mx_scale_value(byte);
  U16x8 v;
  v.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  v.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  v.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  v.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  if (byte == 255u) v.w[0] = v.w[1] = v.w[2] = v.w[3] = 0x7FC07FC0u;
  uint16_t* yr = y + r * K + k;
  if constexpr (VEC) {
    __builtin_nontemporal_store(u32x4{v.w[0], v.w[1], v.w[2], v.w[3]}, reinterpret_cast<u32x4*>(yr));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) yr[j] = static_cast<uint16_t>(v.get(j));
  }
#endif
}

inline bool aligned_to(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// blocks of kMxWaves waves over ceil(M / U) row groups x tiles; 0: too many (a
// launch holds fewer than 2^32 threads, one wave is 64 of them)
unsigned mx_grid(int64_t M, int64_t K, int U) {
  const int64_t groups = (M + U - 1) / U, tiles = mx_tiles(K);
  if (groups > ((1ll << 26) - kMxWaves) / tiles) return 0;
  return static_cast<unsigned>((groups * tiles + kMxWaves - 1) / kMxWaves);
}

template <int ACT>
int launch_quant(const char* what, const uint16_t* x, int64_t ldx, int64_t M, int64_t K, uint8_t* q, uint8_t* s,
                 hipStream_t st) {
  const bool vec = K % 8 == 0 && (M == 1 || ldx % 8 == 0) && aligned_to(x, 16);
  // Four rows per wave once the chip is full of them: more loads in flight per
  // wave (MI355X, us, one row / four: 2080 x 5120 7.3 / 6.6, 8192 x 17408 67 / 58, but
  // 64 x 17408 3.0 / 4.4).
  const int U = M * mx_tiles(K) >= 16384 ? 4 : 1;
  const unsigned grid = mx_grid(M, K, U);
  MW8_REQUIRE(grid > 0, kErrShape, "%s: M=%lld x K=%lld too large", what, (long long)M, (long long)K);
  MW8_REQUIRE(!any_meet({mx_codes_mem(q, M, K), mx_scales_mem(s, M, K)},
                        {RowSet{x, (ACT >= 0 ? 4 : 2) * K, M, 2 * ldx, 1, 0}}),
              kErrArg, "%s: q and s must not overlap each other or x", what);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(kMxThreads), 0, st, x, ldx, M, K, q, s); };
  if (U == 4) {
    if (vec) go(quant_mxfp4_kernel<4, true, ACT>);
    else go(quant_mxfp4_kernel<4, false, ACT>);
  } else {
    if (vec) go(quant_mxfp4_kernel<1, true, ACT>);
    else go(quant_mxfp4_kernel<1, false, ACT>);
  }
  return check_launch(what);
}

}  // namespace

int quant_mxfp4_bf16(const void* x, int64_t M, int64_t K, int64_t ldx, uint8_t* q, uint8_t* s, hipStream_t st) {
  MW8_REQUIRE(x && q && s, kErrArg, "quant_mxfp4: null pointer");
  MW8_REQUIRE(M >= 0 && M < (1ll << 31) && K > 0 && ldx >= K, kErrShape, "quant_mxfp4: bad sizes M=%lld K=%lld ldx=%lld",
              (long long)M, (long long)K, (long long)ldx);
  MW8_REQUIRE(aligned_to(x, 2) && aligned_to(q, 4), kErrAlign, "quant_mxfp4: x needs 2-byte and q 4-byte alignment");
  if (M == 0) return kOk;
  return launch_quant<-1>("quant_mxfp4", static_cast<const uint16_t*>(x), ldx, M, K, q, s, st);
}

int act_and_mul_quant_mxfp4_bf16(const void* x, int64_t R, int64_t two_d, int act, uint8_t* q, uint8_t* s,
                                 hipStream_t st) {
  MW8_REQUIRE(x && q && s, kErrArg, "act_and_mul_quant_mxfp4: null pointer");
  MW8_REQUIRE(act == 0 || act == 1, kErrArg, "act_and_mul_quant_mxfp4: act must be 0 (silu) or 1 (gelu)");
  MW8_REQUIRE(R >= 0 && R < (1ll << 31) && two_d > 0 && two_d % 2 == 0, kErrShape,
              "act_and_mul_quant_mxfp4: bad sizes R=%lld 2d=%lld", (long long)R, (long long)two_d);
  MW8_REQUIRE(aligned_to(x, 2) && aligned_to(q, 4), kErrAlign,
              "act_and_mul_quant_mxfp4: x needs 2-byte and q 4-byte alignment");
  if (R == 0) return kOk;
  const auto* xb = static_cast<const uint16_t*>(x);
  return act == 0 ? launch_quant<0>("act_and_mul_quant_mxfp4", xb, two_d, R, two_d / 2, q, s, st)
                  : launch_quant<1>("act_and_mul_quant_mxfp4", xb, two_d, R, two_d / 2, q, s, st);
}

int dequant_mxfp4_bf16(const uint8_t* q, const uint8_t* s, int64_t M, int64_t K, void* y, hipStream_t st) {
  MW8_REQUIRE(q && s && y, kErrArg, "dequant_mxfp4: null pointer");
  MW8_REQUIRE(M >= 0 && M < (1ll << 31) && K > 0, kErrShape, "dequant_mxfp4: bad sizes M=%lld K=%lld", (long long)M,
              (long long)K);
  MW8_REQUIRE(aligned_to(q, 4) && aligned_to(y, 2), kErrAlign, "dequant_mxfp4: q needs 4-byte and y 2-byte alignment");
  if (M == 0) return kOk;
  const unsigned grid = mx_grid(M, K, 1);
  MW8_REQUIRE(grid > 0, kErrShape, "dequant_mxfp4: M=%lld x K=%lld too large", (long long)M, (long long)K);
  MW8_REQUIRE(!any_meet({one_row(y, M * K * 2)}, {mx_codes_mem(q, M, K), mx_scales_mem(s, M, K)}), kErrArg,
              "dequant_mxfp4: y must not overlap q or s");
  auto* yb = static_cast<uint16_t*>(y);
  if (K % 8 == 0 && aligned_to(y, 16))
    hipLaunchKernelGGL(dequant_mxfp4_kernel<true>, dim3(grid), dim3(kMxThreads), 0, st, q, s, M, K, yb);
  else
    hipLaunchKernelGGL(dequant_mxfp4_kernel<false>, dim3(grid), dim3(kMxThreads), 0, st, q, s, M, K, yb);
  return check_launch("dequant_mxfp4");
}

}  // namespace mw8
