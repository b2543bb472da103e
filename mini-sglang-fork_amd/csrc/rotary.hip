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
#include "row_overlap.h"

namespace mw8 {

namespace {

// Element types by code (the ABI's dtype argument).
template <class T> __device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }

// 1 / rms of a head, as the row norms compute it: the squares of 24-bit values
// are exact in fp64, whose sum hides the order that lanes add in.
__device__ __forceinline__ float norm_factor(double ss, int D, float eps) {
  return 1.0f / __builtin_sqrtf(static_cast<float>(ss / static_cast<double>(D)) + eps);
}

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
    double ss = 0.0;
    for (int i = lane; i < a.D; i += 64) {
      const double v = static_cast<double>(to_f32(x[i]));
      ss = __builtin_fma(v, v, ss);
    }
    for (int off = 32; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
    r = norm_factor(ss, a.D, a.eps);
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

// Whole 16-byte vectors: a lane owns V pairs of a head (V = 8, fp32: 4; two
// vectors, both halves of its pairs), or 2 V elements past the rotated part;
// LPH lanes own a head.  A block takes one token and walks its heads, so a
// lane loads its cosines, sines and norm weights once.  Every element is read
// and written once; the bound is HBM (MI355X: 8000 tokens x 40 heads of 128,
// fp16, 64 rotated, into other tensors 32 us, 5.2 TB/s; in place 27 us; one
// token of 72 heads with norms 3.8 us).
template <class E, bool kInter>
__global__ __launch_bounds__(1024) void rotary_rows_kernel(RotArgs a, int lph) {
  constexpr int V = 16 / sizeof(E);
  struct alignas(16) Vec {
    E e[V];
  };
  const int64_t t = blockIdx.x;
  const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
  if (p < 0) return;  // a padding token: its rows stay as they are
  const int u = threadIdx.x & (lph - 1), heads = a.hq + a.hk, slots = blockDim.x / lph;
  const int half = a.R / 2, turning = half / V;
  const bool turns = u < turning, live = u < a.D / (2 * V);
  // the two vectors' first elements
  const int i0 = kInter || !turns ? 2 * V * u : V * u, i1 = kInter || !turns ? i0 + V : half + V * u;
  float c[V], s[V];
  if (live && turns) {
    const float* cs = a.table + (p < a.P ? p : 0) * a.R + V * u;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c[j] = cs[j];
      s[j] = cs[half + j];
    }
    if (p >= a.P) {  // past the table
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = s[j] = __builtin_nanf("");
    }
  }
  for (int h0 = threadIdx.x / lph; h0 - static_cast<int>(threadIdx.x) / lph < heads; h0 += slots) {
    const bool on = h0 < heads && live;  // (every lane reaches the shuffles)
    const bool is_q = h0 < a.hq;
    const int h = is_q ? h0 : h0 - a.hq;
    const E* x = is_q ? static_cast<const E*>(a.q) + t * a.q_ld + h * a.q_hd : static_cast<const E*>(a.k) + t * a.k_ld + h * a.k_hd;
    E* y = is_q ? static_cast<E*>(a.q_out) + t * a.qo_ld + h * a.qo_hd : static_cast<E*>(a.k_out) + t * a.ko_ld + h * a.ko_hd;
    const E* w = static_cast<const E*>(is_q ? a.qw : a.kw);
    float f0[V], f1[V];
    Vec x0{}, x1{};
    if (on) {
      x0 = *reinterpret_cast<const Vec*>(x + i0);
      x1 = *reinterpret_cast<const Vec*>(x + i1);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f0[j] = to_f32(x0.e[j]);
      f1[j] = to_f32(x1.e[j]);
    }
    if (a.qw || a.kw) {  // launch-uniform
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss = __builtin_fma(static_cast<double>(f0[j]), static_cast<double>(f0[j]), ss);
        ss = __builtin_fma(static_cast<double>(f1[j]), static_cast<double>(f1[j]), ss);
      }
      for (int off = lph / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
      if (on && w) {
        const float r = norm_factor(ss, a.D, a.eps);
        const Vec w0 = *reinterpret_cast<const Vec*>(w + i0), w1 = *reinterpret_cast<const Vec*>(w + i1);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          f0[j] = f0[j] * r * to_f32(w0.e[j]);
          f1[j] = f1[j] * r * to_f32(w1.e[j]);
        }
      }
    }
    if (!on || (!turns && !w && x == y)) continue;
    Vec y0, y1;
    if (!turns) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y0.e[j] = w ? static_cast<E>(f0[j]) : x0.e[j];
        y1.e[j] = w ? static_cast<E>(f1[j]) : x1.e[j];
      }
    } else if constexpr (kInter) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {  // pairs j of the first vector, V / 2 + j of the second
        y0.e[2 * j] = static_cast<E>(f0[2 * j] * c[j] - f0[2 * j + 1] * s[j]);
        y0.e[2 * j + 1] = static_cast<E>(f0[2 * j + 1] * c[j] + f0[2 * j] * s[j]);
        y1.e[2 * j] = static_cast<E>(f1[2 * j] * c[V / 2 + j] - f1[2 * j + 1] * s[V / 2 + j]);
        y1.e[2 * j + 1] = static_cast<E>(f1[2 * j + 1] * c[V / 2 + j] + f1[2 * j] * s[V / 2 + j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y0.e[j] = static_cast<E>(f0[j] * c[j] - f1[j] * s[j]);
        y1.e[j] = static_cast<E>(f1[j] * c[j] + f0[j] * s[j]);
      }
    }
    *reinterpret_cast<Vec*>(y + i0) = y0;
    *reinterpret_cast<Vec*>(y + i1) = y1;
  }
}

// Sine and cosine of p f in fp64: in turns, whose whole part drops exactly.
// The error is p f 2^-53, what rounding the product would leave.
__device__ __forceinline__ void angle_of(double p, double f, double& s, double& c) {
  const double turn = f * 0.15915494309189535;  // / (2 pi)
  const double hi = p * turn, lo = __builtin_fma(p, turn, -hi);
  sincospi(2.0 * ((hi - __builtin_rint(hi)) + lo), &s, &c);
}

// table[p, i] = cos(p f_i) * scale, table[p, R/2 + i] = sin(p f_i) * scale in
// fp64.  A thread fills kTableRows positions from two sines: the next angle
// comes by cos(x + y) = cos x cos y - sin x sin y (the error grows by a few
// 2^-53 a step), 4 multiplications in place of a sine.  Bound: the stores
// (MI355X: 131072 x 128 in 12.9 us, 5.2 TB/s; a sine per element took 33 us).
constexpr int kTableRows = 8;
__global__ __launch_bounds__(256) void rotary_table_kernel(const double* __restrict__ freq, uint32_t half, int64_t P,
                                                           double scale, float* __restrict__ table) {
  const uint32_t n = static_cast<uint32_t>((P + kTableRows - 1) / kTableRows) * half;  // < 2^31 (host)
  for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
    const uint32_t q = e / half, i = e - q * half;
    const int64_t p1 = static_cast<int64_t>(q) * kTableRows;
    const double f = freq[i];
    double s, c, s1, c1;
    angle_of(static_cast<double>(p1), f, s, c);
    angle_of(1.0, f, s1, c1);
    float* row = table + p1 * 2 * half + i;
#pragma unroll
    for (int r = 0; r < kTableRows; ++r) {
      if (p1 + r < P) {
        row[static_cast<int64_t>(2 * r) * half] = static_cast<float>(c * scale);
        row[static_cast<int64_t>(2 * r + 1) * half] = static_cast<float>(s * scale);
      }
      const double cn = __builtin_fma(c, c1, -s * s1);
      s = __builtin_fma(s, c1, c * s1);
      c = cn;
    }
  }
}

// Whether every vector of a tensor's rows is 16-byte aligned.
bool vector_rows(const void* p, int64_t ld, int64_t hd, unsigned size) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * size % 16 == 0 && hd * size % 16 == 0;
}

template <class E>
int launch_rotary(const RotArgs& a, bool inter, hipStream_t st) {
  constexpr unsigned size = sizeof(E);
  constexpr int V = 16 / size;
  const bool vec = a.R % (2 * V) == 0 && a.D % (2 * V) == 0 && a.D <= 128 * V &&
                   (a.hq == 0 || (vector_rows(a.q, a.q_ld, a.q_hd, size) && vector_rows(a.q_out, a.qo_ld, a.qo_hd, size))) &&
                   (a.hk == 0 || (vector_rows(a.k, a.k_ld, a.k_hd, size) && vector_rows(a.k_out, a.ko_ld, a.ko_hd, size))) &&
                   vector_rows(a.qw, 0, 0, size) && vector_rows(a.kw, 0, 0, size) && vector_rows(a.table, 0, 0, 4);
  if (vec) {
    int lph = 1;
    while (lph < a.D / (2 * V)) lph *= 2;
    // few tokens: all of a token's heads at once
    const int most = a.T < 512 ? 1024 : 256, want = (a.hq + a.hk) * lph;
    const unsigned threads = static_cast<unsigned>(want >= most ? most : (want + 63) / 64 * 64);
    if (inter) hipLaunchKernelGGL((rotary_rows_kernel<E, true>), dim3(static_cast<unsigned>(a.T)), dim3(threads), 0, st, a, lph);
    else hipLaunchKernelGGL((rotary_rows_kernel<E, false>), dim3(static_cast<unsigned>(a.T)), dim3(threads), 0, st, a, lph);
    return check_launch("rotary_qk");
  }
  const int64_t rows = a.T * (a.hq + a.hk);
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (inter) hipLaunchKernelGGL((rotary_generic_kernel<E, true>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rotary_generic_kernel<E, false>), dim3(grid), dim3(256), 0, st, a);
  return check_launch("rotary_qk");
}

// Blocks write one token's (or head's) rows while others read theirs, so an
// output may share memory with nothing but the input that it replaces.
int check_rotary_overlap(const RotArgs& a, unsigned size) {
  auto rows = [&](const void* p, int64_t ld, int64_t hd, int heads) {
    const int64_t b = size;
    return RowSet{p, a.D * b, a.T, ld * b, heads, hd * b};
  };
  const RowSet q = rows(a.q, a.q_ld, a.q_hd, a.hq), k = rows(a.k, a.k_ld, a.k_hd, a.hk);
  const RowSet qo = rows(a.q_out, a.qo_ld, a.qo_hd, a.hq), ko = rows(a.k_out, a.ko_ld, a.ko_hd, a.hk);
  auto same = [](const RowSet& x, const RowSet& y) {
    return x.p == y.p && (x.n_outer == 1 || x.outer == y.outer) && (x.n_inner == 1 || x.inner == y.inner);
  };
  MW8_REQUIRE((row_set_empty(qo) || rows_apart(qo)) && (row_set_empty(ko) || rows_apart(ko)), kErrShape,
              "rotary_qk: output rows must not overlap");
  MW8_REQUIRE(!row_sets_meet(qo, ko), kErrArg, "rotary_qk: q_out and k_out must not overlap");
  MW8_REQUIRE((same(qo, q) || !row_sets_meet(qo, q)) && (same(ko, k) || !row_sets_meet(ko, k)), kErrArg,
              "rotary_qk: an output that is not its input must not overlap it");
  MW8_REQUIRE(!row_sets_meet(qo, k) && !row_sets_meet(ko, q), kErrArg, "rotary_qk: q_out and k, k_out and q must not overlap");
  for (const RowSet& r : {one_row(a.pos, a.T * (a.pos64 ? 8 : 4)), one_row(a.table, a.P * a.R * 4),
                          one_row(a.qw, static_cast<int64_t>(a.D) * size), one_row(a.kw, static_cast<int64_t>(a.D) * size)})
    MW8_REQUIRE(!row_sets_meet(qo, r) && !row_sets_meet(ko, r), kErrArg,
                "rotary_qk: the outputs must not overlap positions, table or weights");
  return kOk;
}

}  // namespace

int rotary_qk(const void* q, int64_t q_ld, int64_t q_hd, int hq, const void* k, int64_t k_ld, int64_t k_hd, int hk,
              void* q_out, int64_t qo_ld, int64_t qo_hd, void* k_out, int64_t ko_ld, int64_t ko_hd, int dtype, int D,
              int R, int interleaved, const void* pos, int pos64, const float* table, int64_t P, const void* qw,
              const void* kw, float eps, int64_t T, hipStream_t st) {
  const int64_t heads = static_cast<int64_t>(hq) + hk;
  MW8_REQUIRE(T >= 0 && hq >= 0 && hk >= 0 && heads > 0, kErrShape, "rotary_qk: bad sizes T=%lld heads=%d+%d",
              (long long)T, hq, hk);
  MW8_REQUIRE(D > 0 && D <= 8192 && R > 0 && R <= D && R % 2 == 0, kErrShape,
              "rotary_qk: need an even rotary size in (0, head size <= 8192] (D=%d R=%d)", D, R);
  MW8_REQUIRE(P > 0, kErrShape, "rotary_qk: empty table");
  MW8_REQUIRE(dtype >= 0 && dtype <= 2, kErrArg, "rotary_qk: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  MW8_REQUIRE((hq == 0 || (q && q_out)) && (hk == 0 || (k && k_out)) && pos && table, kErrArg, "rotary_qk: null pointer");
  MW8_REQUIRE(eps >= 0.0f, kErrArg, "rotary_qk: eps must be >= 0");
  if (T == 0) return kOk;
  // (a launch holds fewer than 2^32 threads, here at most 64 per row or 256 per token)
  MW8_REQUIRE(T < (1ll << 24) && T < (1ll << 26) / heads, kErrShape, "rotary_qk: too many rows");
  const unsigned size = dtype == 2 ? 4 : 2;
  auto al = [](const void* p, unsigned b) { return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0; };
  MW8_REQUIRE(al(q, size) && al(k, size) && al(q_out, size) && al(k_out, size) && al(table, 4) && al(pos, pos64 ? 8 : 4) &&
                  al(qw, size) && al(kw, size),
              kErrAlign, "rotary_qk: tensors must be aligned to their elements");
  const RotArgs a{q, k, q_out, k_out, q_ld, q_hd, k_ld, k_hd, qo_ld, qo_hd, ko_ld, ko_hd, pos, table,
                  qw, kw, eps, T, P, hq, hk, D, R, pos64};
  if (const int rc = check_rotary_overlap(a, size)) return rc;
  if (dtype == 0) return launch_rotary<__bf16>(a, interleaved != 0, st);
  if (dtype == 1) return launch_rotary<_Float16>(a, interleaved != 0, st);
  return launch_rotary<float>(a, interleaved != 0, st);
}

int rotary_cos_sin(const double* freq, int half, int64_t P, double scale, float* table, hipStream_t st) {
  MW8_REQUIRE(freq && table, kErrArg, "rotary_cos_sin: null pointer");
  MW8_REQUIRE(half > 0 && half <= 4096 && P >= 0 && P < (1ll << 31) / half, kErrShape,
              "rotary_cos_sin: bad sizes P=%lld pairs=%d", (long long)P, half);
  MW8_REQUIRE((reinterpret_cast<uintptr_t>(freq) & 7u) == 0 && (reinterpret_cast<uintptr_t>(table) & 3u) == 0, kErrAlign,
              "rotary_cos_sin: tensors must be aligned to their elements");
  if (P == 0) return kOk;
  const int64_t blocks = ((P + kTableRows - 1) / kTableRows * half + 255) / 256;
  hipLaunchKernelGGL(rotary_table_kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st,
                     freq, half, P, scale, table);
  return check_launch("rotary_cos_sin");
}

}  // namespace mw8
