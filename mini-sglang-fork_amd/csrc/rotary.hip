// Rotary position embedding of q and k, with the per-head RMSNorm before it,
// and the cos/sin table (gfx950).
//
// A head of D elements turns its first R in R / 2 pairs: element pair i of a
// token at position p becomes (a c - b s, b c + a s) with c = cos[p, i],
// s = sin[p, i].  half layout: pair i is (i, R/2 + i); interleaved: (2i,
// 2i + 1).  With a norm weight the head is first divided by its root mean
// square and multiplied by the weight.  Everything is fp32 between the load
// and the one rounding at the store.
#include "mw8_common.h"

namespace mw8 {

namespace {

// Element types by code (the ABI's dtype argument).
template <class T> __device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }

struct RotArgs {
  const void* q; const void* k;
  void* q_out; void* k_out;
  int64_t q_ld, q_hd, k_ld, k_hd;      // token and head strides of the inputs, elements
  int64_t qo_ld, qo_hd, ko_ld, ko_hd;  // and of the outputs
  const void* pos;
  const float* table;   // [P, R]: R / 2 cosines, then R / 2 sines
  const void* qw; const void* kw;  // norm weights [D] or null
  float eps;
  int64_t T, P;
  int hq, hk, D, R, pos64;
};

// Any layout: one wave per head row.  All of a row's loads for the norm come
// before its stores, and a pair is read and written by one lane, so in-place
// use is safe.
template <class E, bool kInter>
__global__ __launch_bounds__(256) void rotary_generic_kernel(RotArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int heads = a.hq + a.hk;
  if (row >= a.T * heads) return;
  const int64_t t = row / heads;
  int h = static_cast<int>(row - t * heads);
  const bool is_q = h < a.hq;
  if (!is_q) h -= a.hq;
  const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
  if (p < 0) return;  // a padding token: its rows stay as they are
  const E* x = is_q ? static_cast<const E*>(a.q) + t * a.q_ld + h * a.q_hd : static_cast<const E*>(a.k) + t * a.k_ld + h * a.k_hd;
  E* y = is_q ? static_cast<E*>(a.q_out) + t * a.qo_ld + h * a.qo_hd : static_cast<E*>(a.k_out) + t * a.ko_ld + h * a.ko_hd;
  const E* w = static_cast<const E*>(is_q ? a.qw : a.kw);
  float r = 1.0f;
  if (w) {
    float ss = 0.0f;
    for (int i = lane; i < a.D; i += 64) {
      const float v = to_f32(x[i]);
      ss += v * v;
    }
    for (int off = 32; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
    r = 1.0f / __builtin_sqrtf(ss / static_cast<float>(a.D) + a.eps);
  }
  auto in = [&](int i) { return w ? to_f32(x[i]) * r * to_f32(w[i]) : to_f32(x[i]); };
  const int half = a.R / 2;
  const float* cs = a.table + (p < a.P ? p : 0) * a.R;
  for (int i = lane; i < half; i += 64) {
    float c = cs[i], s = cs[half + i];
    if (p >= a.P) c = s = __builtin_nanf("");  // past the table
    const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : half + i;
    const float u = in(ia), v = in(ib);
    y[ia] = static_cast<E>(u * c - v * s);
    y[ib] = static_cast<E>(v * c + u * s);
  }
  if (w || x != y)
    for (int i = a.R + lane; i < a.D; i += 64) y[i] = w ? static_cast<E>(in(i)) : x[i];
}

// table[p, i] = cos(p f_i) * scale, table[p, R/2 + i] = sin(p f_i) * scale,
// the angle and its functions in fp64.
__global__ __launch_bounds__(256) void rotary_table_kernel(const double* __restrict__ freq, int half, int64_t P,
                                                           double scale, float* __restrict__ table) {
  const int64_t n = P * half, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < n; e += step) {
    const int64_t p = e / half;
    const int i = static_cast<int>(e - p * half);
    double s, c;
    sincos(static_cast<double>(p) * freq[i], &s, &c);
    table[p * 2 * half + i] = static_cast<float>(c * scale);
    table[p * 2 * half + half + i] = static_cast<float>(s * scale);
  }
}

template <class E>
int launch_rotary(const RotArgs& a, bool inter, hipStream_t st) {
  const int64_t rows = a.T * (a.hq + a.hk);
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (inter) hipLaunchKernelGGL((rotary_generic_kernel<E, true>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rotary_generic_kernel<E, false>), dim3(grid), dim3(256), 0, st, a);
  return check_launch("rotary_qk");
}

}  // namespace

int rotary_qk(const void* q, int64_t q_ld, int64_t q_hd, int hq, const void* k, int64_t k_ld, int64_t k_hd, int hk,
              void* q_out, int64_t qo_ld, int64_t qo_hd, void* k_out, int64_t ko_ld, int64_t ko_hd, int dtype, int D,
              int R, int interleaved, const void* pos, int pos64, const float* table, int64_t P, const void* qw,
              const void* kw, float eps, int64_t T, hipStream_t st) {
  MW8_REQUIRE(T >= 0 && hq >= 0 && hk >= 0 && hq + hk > 0, kErrShape, "rotary_qk: bad sizes T=%lld heads=%d+%d",
              (long long)T, hq, hk);
  MW8_REQUIRE(D > 0 && D <= 8192 && R > 0 && R <= D && R % 2 == 0, kErrShape,
              "rotary_qk: need an even rotary size in (0, head size <= 8192] (D=%d R=%d)", D, R);
  MW8_REQUIRE(P > 0, kErrShape, "rotary_qk: empty table");
  MW8_REQUIRE(dtype >= 0 && dtype <= 2, kErrArg, "rotary_qk: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  MW8_REQUIRE((hq == 0 || (q && q_out)) && (hk == 0 || (k && k_out)) && pos && table, kErrArg, "rotary_qk: null pointer");
  MW8_REQUIRE(eps >= 0.0f, kErrArg, "rotary_qk: eps must be >= 0");
  if (T == 0) return kOk;
  MW8_REQUIRE(T < (1ll << 31) / (hq + hk), kErrShape, "rotary_qk: too many rows");
  const unsigned size = dtype == 2 ? 4 : 2;
  auto al = [](const void* p, unsigned b) { return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0; };
  MW8_REQUIRE(al(q, size) && al(k, size) && al(q_out, size) && al(k_out, size) && al(table, 4) && al(pos, pos64 ? 8 : 4),
              kErrAlign, "rotary_qk: tensors must be aligned to their elements");
  const RotArgs a{q, k, q_out, k_out, q_ld, q_hd, k_ld, k_hd, qo_ld, qo_hd, ko_ld, ko_hd, pos, table,
                  qw, kw, eps, T, P, hq, hk, D, R, pos64};
  if (dtype == 0) return launch_rotary<__bf16>(a, interleaved != 0, st);
  if (dtype == 1) return launch_rotary<_Float16>(a, interleaved != 0, st);
  return launch_rotary<float>(a, interleaved != 0, st);
}

int rotary_cos_sin(const double* freq, int half, int64_t P, double scale, float* table, hipStream_t st) {
  MW8_REQUIRE(freq && table, kErrArg, "rotary_cos_sin: null pointer");
  MW8_REQUIRE(half > 0 && half <= 4096 && P >= 0 && P < (1ll << 40) / half, kErrShape,
              "rotary_cos_sin: bad sizes P=%lld pairs=%d", (long long)P, half);
  MW8_REQUIRE((reinterpret_cast<uintptr_t>(freq) & 7u) == 0 && (reinterpret_cast<uintptr_t>(table) & 3u) == 0, kErrAlign,
              "rotary_cos_sin: tensors must be aligned to their elements");
  if (P == 0) return kOk;
  const int64_t blocks = (P * half + 255) / 256;
  hipLaunchKernelGGL(rotary_table_kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st,
                     freq, half, P, scale, table);
  return check_launch("rotary_cos_sin");
}

}  // namespace mw8
