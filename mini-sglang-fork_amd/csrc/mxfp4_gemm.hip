// MXFP4 products: y bf16 [M, N] = A W^T of block-scaled 4-bit operands
// (format: mxfp4.h) on v_mfma_scale_f32_16x16x128_f8f6f4.
#include <type_traits>

#include "mxfp4.h"

namespace mw8 {

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct MxArgs {
  const uint8_t* A;   // codes [M, 16 Kb]
  const uint8_t* sa;  // scales [tiles, M, 16]
  const uint8_t* W;   // codes [N, 16 Kb]
  const uint8_t* sw;  // scales [tiles, N, 16]
  const uint16_t* bias;
  uint16_t* out;
  int64_t M, N;
  int kb;     // blocks of 32 along K
  int tiles;  // 512-element tiles along K
};

#if defined(__HIP_DEVICE_COMPILE__)
// D += A B over 128 elements of K; J: the byte of the scale dwords
template <int J>
__device__ __forceinline__ v4f mx_mma(v4i a, v4i b, v4f c, int sa, int sb) {
  const v8i x = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, y = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4 /* e2m1 */, 4, J, sa, J, sb);
}
#endif

// One wave per 16 x 64 output tile, fragments straight from global memory.
__global__ __launch_bounds__(256) void mxfp4_direct_kernel(MxArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kFN = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, grp = lane >> 4;
  const int64_t m0 = (static_cast<int64_t>(blockIdx.y) * 4 + wave) * 16, n0 = static_cast<int64_t>(blockIdx.x) * 16 * kFN;
  if (m0 >= g.M) return;
  const int64_t ld = static_cast<int64_t>(g.kb) * 16;
  const int64_t am = m0 + r16 < g.M ? m0 + r16 : g.M - 1;
  const uint8_t* ap = g.A + am * ld;
  int64_t wn[kFN];
#pragma unroll
  for (int j = 0; j < kFN; ++j) wn[j] = n0 + 16 * j + r16 < g.N ? n0 + 16 * j + r16 : g.N - 1;
  v4f acc[kFN] = {};
  for (int t = 0; t < g.tiles; ++t) {
    const int sa = *reinterpret_cast<const int*>(g.sa + (t * g.M + am) * 16 + 4 * grp);
    int sw[kFN];
#pragma unroll
    for (int j = 0; j < kFN; ++j) sw[j] = *reinterpret_cast<const int*>(g.sw + (t * g.N + wn[j]) * 16 + 4 * grp);
    auto step = [&](auto jc) {
      constexpr int J = decltype(jc)::value;
      int c = 16 * t + 8 * (J >> 1) + 2 * grp + (J & 1);
      c = c < g.kb ? c : g.kb - 1;  // blocks past K: their scales are 2^-127 on both sides
      const v4i a = *reinterpret_cast<const v4i*>(ap + 16 * c);
#pragma unroll
      for (int j = 0; j < kFN; ++j) {
        const v4i w = *reinterpret_cast<const v4i*>(g.W + wn[j] * ld + 16 * c);
        acc[j] = mx_mma<J>(a, w, acc[j], sa, sw[j]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int j = 0; j < kFN; ++j) {
    const int64_t n = n0 + 16 * j + r16;
    if (n >= g.N) continue;
    const float b = g.bias ? bf16_to_f32(g.bias[n]) : 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t m = m0 + 4 * grp + v;
      if (m < g.M) g.out[m * g.N + n] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(acc[j][v] + b));
    }
  }
#endif
}

inline bool aligned_to(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace

int gemm_mxfp4_bf16(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, const void* bias, void* y,
                    int64_t M, int64_t N, int64_t K, hipStream_t st) {
  MW8_REQUIRE(A && sa && W && sw && y, kErrArg, "gemm_mxfp4: null pointer");
  MW8_REQUIRE(M >= 0 && N > 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K <= (1ll << 20), kErrShape,
              "gemm_mxfp4: bad sizes M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  MW8_REQUIRE(aligned_to(A, 16) && aligned_to(W, 16) && aligned_to(sa, 16) && aligned_to(sw, 16), kErrAlign,
              "gemm_mxfp4: A, sa, W and sw need 16-byte alignment");
  if (M == 0) return kOk;
  const MxArgs g{A, sa, W, sw, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(y), M, N,
                 static_cast<int>(mx_blocks(K)), static_cast<int>(mx_tiles(K))};
  const int64_t gy = (M + 63) / 64, gx = (N + 63) / 64;
  MW8_REQUIRE(gy < 65536, kErrShape, "gemm_mxfp4: M=%lld too large", (long long)M);
  hipLaunchKernelGGL(mxfp4_direct_kernel, dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(256), 0, st, g);
  return check_launch("gemm_mxfp4");
}

}  // namespace mw8
