// MXFP4 products for few tokens: the weights stream once, K split over the
// waves of a block, or, for many weight rows, the rows.
#pragma once

#include "mxfp4_ring.h"

namespace mw8 {

struct MxDecodeArgs {
  MxArgs g;
  const uint16_t* x;  // kXQ: bf16 rows [M, ldx] in place of g.A / g.sa
  int64_t ldx, K;
  int per_wave;  // 512-element tiles per wave
};

namespace {

// kXQ: rows x tiles that a wave quantizes.  A pass costs a wave some 0.15 us
// that every block pays: the launch that it saves is worth 8 (MI355X, us,
// one launch / two: 2 x 5120 -> 7168 7.2 / 8.3, 4 rows 8.7 / 8.4; 4 x 2048 ->
// 5120 5.1 / 6.3).
constexpr int kMxPasses = 8;
constexpr int kMxSlot = 4096;  // 16 weight rows x 256 code bytes (RG of them per tile)

// Block b owns weight rows [N b / G, N (b + 1) / G), at most 16 RG of them,
// so a grid of a multiple of the CU count gives every CU the same bytes.  Wave
// w takes 512-element tiles [w per_wave, (w + 1) per_wave) of K: the codes
// of a tile (256 contiguous bytes of each row, 1 KB per instruction) go into
// a private ring of D slots by DMA, its scales (256 contiguous bytes per 16
// rows) and the tokens' codes and scales into registers.  Four matrix
// instructions per 16 rows use a tile, weight rows as their rows, 16 tokens
// as columns.  No barrier before the end; the waves' fp32 sums are then added
// in wave order.  Bound: HBM, every weight byte read once.  MI355X, weights
// from HBM: 1 x 51200 x 5120 24.1 us (5.8 TB/s, what a streaming read
// reaches), 1 x 34816 x 5120 17.6 us, 1 x 5120 x 17408 11.2 us, 1 x 7168 x
// 5120 5.8 us (launch, first loads and last sums are some 3 us of each).
//
// kXQ: the tokens are bf16 rows, quantized by the wave that multiplies them
// (its own part of K only): one pass per row and tile, 8 elements per lane,
// codes and scales through LDS.
template <int RG, int D, bool kXQ>
__global__ __launch_bounds__(1024) void mxfp4_decode_kernel(MxDecodeArgs d) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kOps = 5 * RG + (kXQ ? 0 : 5);  // vector memory operations per tile
  static_assert((D - 1) * kOps < 64, "ring depth");
  constexpr int kSlot = RG * kMxSlot;
  const MxArgs& g = d.g;
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, grp = lane >> 4;
  const int64_t n0 = g.N * blockIdx.x / gridDim.x;
  const int rows = static_cast<int>(g.N * (blockIdx.x + 1) / gridDim.x - n0);
  if (rows <= 0) return;
  const int M = static_cast<int>(g.M);
  const int64_t ld = static_cast<int64_t>(g.kb) * 16;
  const int t0 = wave * d.per_wave, t1 = t0 + d.per_wave < g.tiles ? t0 + d.per_wave : g.tiles;
  unsigned char* ring = lds + wave * (D * kSlot);
  unsigned char* xq = lds + waves * (D * kSlot) + static_cast<int64_t>(t0) * (M * 272);  // kXQ: [tile][row][256 + 16]

  auto view = [](const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(scalar_ptr(const_cast<uint8_t*>(static_cast<const uint8_t*>(p))), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kBufferFlags);
  };
  const __amdgpu_buffer_rsrc_t w_rsrc = view(g.W + n0 * ld, rows * ld);
  const __amdgpu_buffer_rsrc_t a_rsrc = view(kXQ ? nullptr : g.A, kXQ ? 0 : M * ld);
  // DMA instruction j: rows 4 j .. 4 j + 3, chunk c of row r at c ^ r
  uint32_t w_off[4 * RG];
#pragma unroll
  for (int j = 0; j < 4 * RG; ++j) {
    const int row = 4 * j + grp;
    w_off[j] = static_cast<uint32_t>(row * ld + 16 * (r16 ^ (row & 15)));
  }
  int sw[D][RG], sa[D];
  v4i xa[kXQ ? 1 : D][4];
  auto issue = [&](int slot, int t) {
    const bool live = t < t1;  // else: out of every view's range (zeros, no traffic)
    const int koff = live ? t * 256 : 0x7fff0000;
#pragma unroll
    for (int j = 0; j < 4 * RG; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, (lds_ptr_t)(ring + slot * kSlot + j * 1024), 16, w_off[j], koff, 0,
                                               kStreamAux);
    const int64_t tt = live ? t : 0;
    const __amdgpu_buffer_rsrc_t sw_rsrc = view(g.sw + (tt * g.N + n0) * 16, live ? rows * 16 : 0);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
      sw[slot][rg] = __builtin_amdgcn_raw_buffer_load_b32(sw_rsrc, (16 * rg + r16) * 16 + 4 * grp, 0, 0);
    if constexpr (!kXQ) {
      const __amdgpu_buffer_rsrc_t s_rsrc = view(g.sa + tt * M * 16, live ? M * 16 : 0);
      sa[slot] = __builtin_amdgcn_raw_buffer_load_b32(s_rsrc, r16 * 16 + 4 * grp, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xa[slot][j] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
            a_rsrc, static_cast<uint32_t>(r16 * ld + 16 * (8 * (j >> 1) + 2 * grp + (j & 1))), koff, 0));
    }
  };
  v4f acc[RG] = {};
  auto consume = [&](int slot, int t) {
    if constexpr (kXQ) sa[slot] = *reinterpret_cast<const int*>(xq + ((t - t0) * M + (r16 < M ? r16 : 0)) * 272 + 256 + 4 * grp);
    auto step = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      const int c = 8 * (j >> 1) + 2 * grp + (j & 1);
      v4i a;
      if constexpr (kXQ) {
        const int r = r16 < M ? r16 : 0;
        a = *reinterpret_cast<const v4i*>(xq + ((t - t0) * M + r) * 272 + 16 * (c ^ r));
      } else {
        a = xa[slot][j];
      }
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const v4i w = *reinterpret_cast<const v4i*>(ring + slot * kSlot + rg * kMxSlot + r16 * 256 + 16 * (c ^ r16));
        acc[rg] = mx_mma<j>(w, a, acc[rg], sw[slot][rg], sa[slot]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  };

  if constexpr (kXQ) {
    // tokens in passes of one row and tile (8 elements a lane), at most
    // kMxPasses, loaded ahead of the weights of the first D tiles and
    // quantized under these
    const __amdgpu_buffer_rsrc_t x_rsrc = view(d.x, ((M - 1) * d.ldx + d.K) * 2);
    const int passes = (t1 - t0) * M;
    U16x8 v[kMxPasses];
    int t = t0, r = 0;
#pragma unroll
    for (int u = 0; u < kMxPasses; ++u) {
      const int64_t k = static_cast<int64_t>(t) * 512 + 8 * lane;
      const uint32_t off = u < passes && k < d.K ? static_cast<uint32_t>((r * d.ldx + k) * 2) : 0x80000000u;
      const auto q = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, off, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[u].w[j] = q[j];
      if (++r == M) {
        r = 0;
        ++t;
      }
    }
#pragma unroll
    for (int s = 0; s < D; ++s) issue(s, t0 + s);
    r = 0;
#pragma unroll
    for (int u = 0; u < kMxPasses; ++u) {
      if (u >= passes) break;  // wave-uniform
      uint32_t byte;
      const uint32_t codes = mx_quant_quad(v[u], byte);
      unsigned char* row = xq + u * 272;
      *reinterpret_cast<uint32_t*>(row + 16 * ((lane >> 2) ^ r) + 4 * (lane & 3)) = codes;
      if ((lane & 3) == 0) row[256 + mx_scale_pos(lane >> 2)] = static_cast<unsigned char>(byte);
      if (++r == M) r = 0;
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // this wave's LDS writes (it alone reads them)
  } else {
#pragma unroll
    for (int s = 0; s < D; ++s) issue(s, t0 + s);
  }
  const int n_pad = (t1 - t0 + D - 1) / D * D;
  int t = t0;
  for (; t < t0 + n_pad - D; t += D) {
#pragma unroll
    for (int s = 0; s < D; ++s) {
      wait_vmcnt<(D - 1) * kOps>();
      consume(s, t + s);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // the slot's fragments are read before its refill
      issue(s, t + s + D);
    }
  }
  if (t1 > t0) {
    auto last = [&](auto sc) {
      constexpr int s = decltype(sc)::value;
      if constexpr (s < D) {
        wait_vmcnt<(D - 1 - s) * kOps>();
        if (t + s < t1) consume(s, t + s);
      }
    };
    last(std::integral_constant<int, 0>{});
    last(std::integral_constant<int, 1>{});
    last(std::integral_constant<int, 2>{});
    last(std::integral_constant<int, 3>{});
    last(std::integral_constant<int, 4>{});
    last(std::integral_constant<int, 5>{});
  }
  wait_vmcnt<0>();
  __syncthreads();  // the ring becomes the waves' sums: [wave][16 tokens][16 RG rows + 1]
  float* red = reinterpret_cast<float*>(lds);
  constexpr int kRow = 16 * RG + 1, kSum = 16 * kRow;
#pragma unroll
  for (int rg = 0; rg < RG; ++rg)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave * kSum + r16 * kRow + 16 * rg + 4 * grp + v] = acc[rg][v];
  __syncthreads();
  for (int e = tid; e < 256 * RG; e += blockDim.x) {
    const int m = e / (16 * RG), n = e % (16 * RG);
    if (m >= M || n >= rows) continue;
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += red[w * kSum + m * kRow + n];
    if (g.bias) s += bf16_to_f32(g.bias[n0 + n]);
    g.out[m * g.N + n0 + n] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(s));
  }
#endif
}

// Many weight rows: one block per CU keeps the tokens in LDS ([tile][16 TG
// rows][256 code bytes, chunk c of row r at c ^ r], then scales [tile][16 TG
// rows][16]).  It owns weight rows in units of 4; its waves split them evenly and
// walk them in chunks of at most 16 rows, all of K each, through private rings
// of D slots, so no sum crosses waves and nothing is synchronized after the
// start.  (Above, every block loads the tokens again, 16 bytes a cycle where the
// lanes of a load lie on different rows: 16 tokens cost 4 us more than one at
// 34816 x 5120.)  Bound: HBM.  MI355X: 16 x 34816 x 5120 18.3 us (5.2 TB/s; split
// along K 21.7), 32 tokens 19.0 (64 x 64 ring 25.3); 16 x 51200 x 5120 25.2 us
// (5.5 TB/s; 29.3), 32 tokens 26.4 (35.1).
template <int TG, int D>
__global__ __launch_bounds__(1024) void mxfp4_decode_shared_kernel(MxArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kOps = 5;  // vector memory operations per tile
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, grp = lane >> 4, waves = blockDim.x >> 6;
  const int64_t units = (g.N + 3) / 4, parts = static_cast<int64_t>(gridDim.x) * waves;
  const int64_t part = static_cast<int64_t>(blockIdx.x) * waves + wave;
  const int64_t u0 = units * part / parts, u1 = units * (part + 1) / parts;
  const int own = static_cast<int>(u1 - u0), chunks = (own + 3) / 4;
  const int M = static_cast<int>(g.M), tiles = g.tiles;
  const int64_t ld = static_cast<int64_t>(g.kb) * 16;
  unsigned char* const tok = lds;
  unsigned char* const tok_s = lds + tiles * (TG * kMxSlot);
  unsigned char* const ring = tok_s + tiles * (TG * 256) + wave * (D * kMxSlot);
  auto view = [](const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(scalar_ptr(const_cast<uint8_t*>(static_cast<const uint8_t*>(p))), 0,
                                             __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kBufferFlags);
  };
  uint32_t off[4];  // DMA instruction j: rows 4 j .. 4 j + 3, chunk c of row r at c ^ r
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = 4 * j + grp;
    off[j] = static_cast<uint32_t>(row * ld + 16 * (r16 ^ row));
  }
  // chunk c of the wave: units [u0 + own c / chunks, u0 + own (c + 1) / chunks)
  auto first = [&](int c) { return 4 * (u0 + static_cast<uint32_t>(own * c) / static_cast<uint32_t>(chunks)); };
  // the next tile to load: tile it of chunk ic, weight rows n_in .. n_in + rows - 1
  // (none behind the last chunk: every load reads zeros)
  int ic = 0, it = 0, rows = 0;
  int64_t n_in = 0;
  auto enter = [&] {
    const bool live = ic < chunks;
    const int64_t end = live ? first(ic + 1) : 0;
    n_in = live ? first(ic) : 0;
    rows = static_cast<int>((end < g.N ? end : g.N) - n_in);
  };
  enter();
  int sw[D];
  auto issue = [&](int slot) {
    const __amdgpu_buffer_rsrc_t w_rsrc = view(g.W + n_in * ld, rows * ld);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, (lds_ptr_t)(ring + slot * kMxSlot + j * 1024), 16, off[j], it * 256, 0,
                                               kStreamAux);
    const __amdgpu_buffer_rsrc_t sw_rsrc = view(g.sw + (it * g.N + n_in) * 16, rows * 16);
    sw[slot] = __builtin_amdgcn_raw_buffer_load_b32(sw_rsrc, r16 * 16 + 4 * grp, 0, 0);
    if (++it == tiles) {
      it = 0;
      ++ic;
      enter();
    }
  };
  const __amdgpu_buffer_rsrc_t a_rsrc = view(g.A, M * ld);
  for (int t = wave; t < tiles; t += waves) {
#pragma unroll
    for (int tg = 0; tg < TG; ++tg)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (lds_ptr_t)(tok + (t * TG + tg) * kMxSlot + j * 1024), 16,
                                                 static_cast<uint32_t>(off[j] + 16 * tg * ld), t * 256, 0, 0);
    const __amdgpu_buffer_rsrc_t s_rsrc = view(g.sa + static_cast<int64_t>(t) * M * 16, M * 16);
    if (lane < 16 * TG) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(s_rsrc, lane * 16, 0, 0);
      *reinterpret_cast<v4i*>(tok_s + t * (TG * 256) + lane * 16) = __builtin_bit_cast(v4i, v);
    }
  }
#pragma unroll
  for (int s = 0; s < D; ++s) issue(s);
  wait_vmcnt<D * kOps>();  // this wave's part of the tokens
  __syncthreads();
  v4f acc[TG] = {};
  int c = 0, t = 0;
  auto consume = [&](int slot) {
    const unsigned char* const ws = ring + slot * kMxSlot + r16 * 256;
    v4i w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const v4i*>(ws + 16 * ((8 * (j >> 1) + 2 * grp + (j & 1)) ^ r16));
#pragma unroll
    for (int tg = 0; tg < TG; ++tg) {
      const unsigned char* const xs = tok + (t * TG + tg) * kMxSlot + r16 * 256;
      const int s = *reinterpret_cast<const int*>(tok_s + (t * TG + tg) * 256 + r16 * 16 + 4 * grp);
      v4i x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const v4i*>(xs + 16 * ((8 * (j >> 1) + 2 * grp + (j & 1)) ^ r16));
      acc[tg] = mx_mma<0>(w[0], x[0], acc[tg], sw[slot], s);
      acc[tg] = mx_mma<1>(w[1], x[1], acc[tg], sw[slot], s);
      acc[tg] = mx_mma<2>(w[2], x[2], acc[tg], sw[slot], s);
      acc[tg] = mx_mma<3>(w[3], x[3], acc[tg], sw[slot], s);
    }
  };
  auto finish = [&] {  // chunk c is summed: a lane holds 4 columns of token r16
    const int64_t n0 = first(c) + 4 * grp, end = first(c + 1), n1 = end < g.N ? end : g.N;
    if (n0 < n1) {
#pragma unroll
      for (int tg = 0; tg < TG; ++tg) {
        const int m = 16 * tg + r16;
        uint16_t o[4];
#pragma unroll
        for (int v = 0; v < 4; ++v)
          o[v] = __builtin_bit_cast(
              uint16_t, static_cast<__bf16>(acc[tg][v] + (g.bias && n0 + v < n1 ? bf16_to_f32(g.bias[n0 + v]) : 0.0f)));
        uint16_t* at = g.out + m * g.N + n0;
        if (m < M) {
          if (g.store >= 4) {
            *reinterpret_cast<uint2*>(at) = make_uint2(o[0] | static_cast<uint32_t>(o[1]) << 16, o[2] | static_cast<uint32_t>(o[3]) << 16);
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (n0 + v < n1) at[v] = o[v];
          }
        }
      }
    }
#pragma unroll
    for (int tg = 0; tg < TG; ++tg) acc[tg] = v4f{};
  };
  const int items = chunks * tiles;
  for (int i = 0; i < items; i += D) {
#pragma unroll
    for (int s = 0; s < D; ++s) {
      wait_vmcnt<(D - 1) * kOps>();  // (loads retire in order; a chunk's stores only make it wait for more)
      if (i + s < items) {
        consume(s);
        if (++t == tiles) {
          finish();
          t = 0;
          ++c;
        }
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // the slot's fragments are read before its refill
      issue(s);
    }
  }
  wait_vmcnt<0>();
#endif
}

}  // namespace
}  // namespace mw8
