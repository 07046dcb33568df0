// Microscaled 4-bit matrices (MX4) and the linear product with them, for serving a model whose weights are held in
// 4 bits.  The reference has no counterpart (its models run in bf16 and fp32).
//
// A row of K elements is held as G = ceil(K / 128) groups of 128: 64 bytes of codes (two E2M1 elements to a byte, the
// lower nibble first) and 4 scale bytes.  32 consecutive elements share the scale s, which stands for 2^(s - 127)
// (255: the block is NaN).  The padding past K is zero, so a product runs over whole groups.
#include "kdn_common.h"
#include "kdn_state.h"
#include "../../include/kdn.h"

namespace {

using kdn_state::mfma;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------
// Quantisation.  With E the exponent field of the block's largest magnitude, s = max(E - 2, 0) (so that magnitude
// lies in [4, 8) units of 2^(s - 127)) and every element is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6
// units, ties to the even code, larger ones to 6.  A block that holds an infinity or NaN gets s = 255.
// A lane takes 8 elements, four lanes a block.  Bound by the bytes: 14416 x 2304 bf16 17.1 us (4.9 TB/s), back 13.0; 1999 x
// 7208 fp32 11.1 and 13.9 (4.7 TB/s; with 8 fp32 a lane, every second 16 bytes to a store, 17.7).  A matrix whose rows
// start anywhere takes the same wide accesses (element by element, quantising and back 1999 x 7207 bf16 took 41 us, now 18).
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = load16(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) v[2 * q] = __uint_as_float(w[q] << 16), v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    } else {
      *reinterpret_cast<uint4*>(v) = load16(p);
      *reinterpret_cast<uint4*>(v + 4) = load16(p + 4);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? ld<T>(p, e) : 0.f;
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ x, int64_t xs, int K, uint32_t per,
                                                           uint32_t items, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= items) return;  // items is a multiple of 16: whole quads
  const uint32_t row = i / per, seg = i - row * per;
  float v[8];
  load8(x + (int64_t)row * xs + 8 * seg, K - (int)(8 * seg), v);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, kDppXor1, 0xF, 0xF, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, kDppXor2, 0xF, 0xF, false));
  const uint32_t field = top >> 23, s = field == 255 ? 255u : (field > 2 ? field - 2 : 0u);
  const float unit = __uint_as_float(s << 23);  // the conversion reads the exponent field alone (0: 2^-127)
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], unit, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], unit, 3);
  codes[i] = s == 255 ? 0u : c;
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
}

// 16 bytes of values per lane (8 bf16, 4 fp32); every value of MX4 is a bf16 number
template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int K,
                                                             uint32_t per, uint32_t items, T* __restrict__ y) {
  constexpr int E = 16 / sizeof(T);
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= items) return;
  const uint32_t row = i / per, seg = i - row * per;
  const int n = K - (int)(E * seg);
  if (n <= 0) return;
  const uint32_t c = E == 8 ? reinterpret_cast<const uint32_t*>(codes)[i] : reinterpret_cast<const uint16_t*>(codes)[i];
  const float unit = __uint_as_float((uint32_t)scales[i / (32 / E)] << 23);
  uint32_t w[4];
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 0));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 1));
  if constexpr (E == 8) {
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 2));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 3));
  } else {
    w[3] = w[1] & 0xffff0000u, w[2] = w[1] << 16, w[1] = w[0] & 0xffff0000u, w[0] <<= 16;
  }
  T* p = y + (int64_t)row * K + E * seg;
  if (n >= E) {
    store16(p, uint4{w[0], w[1], w[2], w[3]});
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (e >= n) continue;
    if constexpr (E == 8)
      reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
    else
      reinterpret_cast<uint32_t*>(p)[e] = w[e];
  }
}

// ---------------------------------------------------------------------------------------------
// y[m, n] = epilogue(sum_k x[m, k] W[n, k]): + bias; GATED (W = [W1; W2]): silu(W1 x + b1) (W2 x + b2); + res[m, n],
// in fp32 before the one rounding to bf16.  x is bf16 (W's elements are bf16 numbers, so the bf16 products are those
// of the dequantised weights) or MX4 (XQ: the scaled 4-bit products of the matrix cores).
// ---------------------------------------------------------------------------------------------
struct MxArgs {
  const uint8_t *x, *xsc;
  int64_t xs;  // bf16 x: row stride in elements
  const uint8_t *W, *wsc;
  const bf16_t *bias, *res;
  int64_t rs;
  int M, N, K, G;
  bf16_t* y;
  int64_t ys;
};

__device__ __forceinline__ uint32_t deq2(uint32_t c, float unit, int sel) {
  switch (sel) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, unit, 3));
  }
}
// 8 codes -> 8 bf16
__device__ __forceinline__ uint4 deq8(uint32_t c, float unit) {
  return uint4{deq2(c, unit, 0), deq2(c, unit, 1), deq2(c, unit, 2), deq2(c, unit, 3)};
}

__device__ __forceinline__ i32x8 codes8(uint4 c) { return i32x8{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0}; }
__device__ __forceinline__ uint4 buf_ld16(bufrsrc r, uint32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
constexpr uint32_t kOut = 0x80000000u;  // a buffer offset past every buffer: loads 0

// silu(a) b; e^-a = inf for very negative a gives -0.  (The hardware's reciprocal and exponential, about 2^-22 off, before
// a rounding to 8 bits: an IEEE division made the epilogue of 2304-element sums a quarter of the product's time.)  The
// reciprocal flushes subnormal results, so it is taken of a quarter of 1 + e^-a, at most 2^126 or infinite.
__device__ __forceinline__ float mx_gate(float a, float b) {
  return 0.25f * a * frcp(__builtin_fmaf(fexp(-a), 0.25f, 0.25f)) * b;
}
// One output of the epilogue, from the sum of W's row n (and, gated, of W2's).
__device__ __forceinline__ float mx_epilogue(const MxArgs& A, int m, int n, float v0, float v1, bool gated) {
  float o = v0 + (A.bias ? bf2f(A.bias[n]) : 0.f);
  if (gated) o = mx_gate(o, v1 + (A.bias ? bf2f(A.bias[A.N + n]) : 0.f));
  if (A.res) o += bf2f(A.res[(int64_t)m * A.rs + n]);
  return o;
}

// Loads from a buffer straight to LDS: 64 lanes' 16 bytes to `lds` (uniform, an LDS address) and on; a lane whose
// offset lies past the buffer writes 0.  In assembler because the compiler, which can not tell the two stages' buffers
// apart, would wait for the loads in flight before every read of the other one; they have no output registers, are
// waited for by dma_wait, and leave the compiler's own counts too strict, never too lax.  M0 needs one wait state.
__device__ __forceinline__ u32x4 dma_buf(const void* base, uint32_t bytes) {  // uniform
  const uint64_t a = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ void dma16(u32x4 r, uint32_t lds, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(voff), "s"(r), "s"(__builtin_amdgcn_readfirstlane(soff))
               : "m0", "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A row's pieces of 16 bytes lie in LDS at c ^ turn(row).  A 16-byte read serves lanes 0-3, 12-15 and 20-27 in one go, then
// 4-11, 16-19 and 28-31 (and likewise the upper half), so lane (r, kg)'s rows 4 to 11 meet rows 0-3 and 12-15 of its
// neighbour kg; these turns put all sixteen into different banks (turning by r alone, half of them met another).
template <int CH>
__device__ __forceinline__ int turn(int row) {
  if (CH == 16) return (row + 12) & 15;
  if (CH == 8) return ((row >> 1) + 6) & 7;
  return (((row >> 2) ^ (row >> 3)) & 1) << 1 | (row >> 2 & 1);  // CH 4
}

// ---- at most 16 rows of x -----------------------------------------------------------------------------------------
// Bound by the weight stream: every byte of W is read once, straight into the matrix cores' operand layout (lane
// (r, kg) holds row r's block kg of a group, 16 bytes), and converted to bf16 there (one instruction for two
// elements); x's rows are the other operand (the columns past M unused).  The 8 waves of a workgroup split the groups
// of K and meet in LDS; the workgroup walks tiles of `tr` rows of W, the next tile's loads in flight meanwhile.
// bf16 x lies in LDS (loaded in the operand layout, four neighbouring lanes in four rows, M 8, K 7208 took 14000
// accesses to L1 per workgroup); MX4 x, a quarter of that, in registers.  SW: groups per wave and chunk of K.  K past 8 SW
// groups, or more of x than LDS holds, is walked in chunks of two buffers, x read again for every tile.
// Gated N 7208, K 2304, M 1 to 8: 7.1 to 7.5 us (2.5 TB/s of W), M 16 8.7; N 2304, K 7208: M 1 5.4, M 4 5.7, M 8 6.7, M 16 (x
// in four chunks) 11.7.  The waves spend half of the time in waits: a few rounds of latency (launch, W's first loads, the
// meeting in LDS), of which more loads in flight took nothing, and at a long K from 8 rows on also x, all of which every
// workgroup loads before its first product.
constexpr int kFewWaves = 8, kFewLds = 131072;

template <bool XQ, int NA, int SW>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_linear_few_kernel(const MxArgs A, int tr, int tiles, int chunks, int over_m,
                                                                              int half) {
  constexpr int NW = kFewWaves, T = 64 * NW, SQ = (SW + 3) / 4;
  __shared__ float s_acc[2][NW][NA][256];
  extern __shared__ uint4 s_few[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kg = lane >> 4, G = A.G, M = A.M;
  const uint32_t wrow = (uint32_t)G * 64, srow = (uint32_t)G * 4;
  struct Wt {
    uint4 c[SW][NA];
    uint4 s[SQ][NA];  // the scales of four groups in a row
  };
  struct Xq {
    uint4 c[XQ ? SW : 1];
    uint32_t s[XQ ? SW : 1];
  };
  // chunk c is the groups [from(c), from(c + 1)); this wave's of it begin at first(c, wv) and end at first(c, wv + 1)
  auto from = [&](int c) { return (int)((int64_t)G * c / chunks); };
  auto first = [&](int c, int w) { return from(c) + (from(c + 1) - from(c)) * w / NW; };
  const int xm = min(r, M - 1);
  const bufrsrc rx = make_buf(A.x, XQ ? (uint32_t)M * wrow : 0u), rxs = make_buf(A.xsc, XQ ? (uint32_t)M * srow : 0u);
  const u32x4 dx = dma_buf(A.x, XQ ? 0u : (uint32_t)(((int64_t)(M - 1) * A.xs + A.K) * 2));
  auto load_x = [&](Xq& x, int c, int buf) {
    if constexpr (XQ) {
      const int g0 = first(c, wv), g1 = first(c, wv + 1);
#pragma unroll
      for (int u = 0; u < SW; ++u) {
        x.c[u] = buf_ld16(rx, g0 + u < g1 ? (uint32_t)xm * wrow + 64u * (g0 + u) + 16 * kg : kOut);
        x.s[u] = __builtin_amdgcn_raw_buffer_load_b8(rxs, g0 + u < g1 ? (uint32_t)xm * srow + 4u * (g0 + u) + kg : kOut, 0, 0);
      }
    } else {
      // all of the chunk: [group][row][16 pieces at c ^ turn(row)], 512 pieces at a time (the last ones past it: 0)
      const int b = from(c), rows = (from(c + 1) - b) * M;
      for (int q = 0; q < rows * 16; q += T) {
        const int at = (q + tid) >> 4, g = (at * over_m) >> 16, row = at - g * M, k = 128 * (b + g) + 8 * ((tid & 15) ^ turn<16>(row));
        dma16(dx, lds_address(s_few + buf * half + q + 64 * wv), at < rows && k < A.K ? ((uint32_t)row * (uint32_t)A.xs + k) * 2 : kOut, 0u);
      }
    }
  };
  auto load_w = [&](Wt& w, int tile, int c) {
    const int g0 = first(c, wv), g1 = first(c, wv + 1), n0 = tile * tr, rows = min(tr, A.N - n0);
#pragma unroll
    for (int a = 0; a < NA; ++a) {  // rows past the tile's are 0 (and not read)
      const int64_t row = (int64_t)a * A.N + n0;
      const bufrsrc rw = make_buf(A.W + row * wrow, (uint32_t)rows * wrow), rs = make_buf(A.wsc + row * srow, (uint32_t)rows * srow);
      const uint32_t vw = (uint32_t)r * wrow + 64u * g0 + 16 * kg, vs = (uint32_t)r * srow + 4u * g0;
#pragma unroll
      for (int u = 0; u < SW; ++u) w.c[u][a] = buf_ld16(rw, g0 + u < g1 ? vw + 64u * u : kOut);
#pragma unroll
      for (int q = 0; q < SQ; ++q) w.s[q][a] = buf_ld16(rs, vs + 16u * q);  // (scales of groups that are not used may follow)
    }
  };
  f32x4 acc[NA];
  auto compute = [&](const Wt& w, const Xq& x, int c, int buf) {
    const int g0 = first(c, wv), g1 = first(c, wv + 1);
#pragma unroll
    for (int u = 0; u < SW; ++u) {
      if (g0 + u >= g1) break;  // uniform
      uint4 xf[4];
      if constexpr (!XQ) {
        const uint4* p = s_few + buf * half + ((g0 + u - from(c)) * M + xm) * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[j] = p[(4 * kg + j) ^ turn<16>(xm)];
      }
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        const uint4 sq = w.s[u / 4][a];
        const uint32_t s = ((u & 3) == 0 ? sq.x : (u & 3) == 1 ? sq.y : (u & 3) == 2 ? sq.z : sq.w) >> (8 * kg) & 255u;
        if constexpr (XQ) {
          acc[a] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes8(w.c[u][a]), codes8(x.c[u]), acc[a], 4, 4, 0, s, 0, x.s[u]);
        } else {
          const float unit = __uint_as_float(s << 23);
          acc[a] = mfma(deq8(w.c[u][a].x, unit), xf[0], acc[a]);
          acc[a] = mfma(deq8(w.c[u][a].y, unit), xf[1], acc[a]);
          acc[a] = mfma(deq8(w.c[u][a].z, unit), xf[2], acc[a]);
          acc[a] = mfma(deq8(w.c[u][a].w, unit), xf[3], acc[a]);
        }
      }
    }
  };
  Wt w, next;
  Xq x, xn;
  load_w(w, blockIdx.x, 0);
  load_x(x, 0, 0);
  dma_wait();
  __syncthreads();
  int buf = 0, xb = 0;
  bool fresh = false;  // the step's loads are in `next` (taken at its start: they fly during the sums before it)
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
#pragma unroll
    for (int a = 0; a < NA; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < chunks; ++c) {
      if (fresh) {
        w = next;
        if (chunks > 1) {
          x = xn, xb ^= 1;
          dma_wait();
          __syncthreads();
        }
      }
      const int tn = c + 1 < chunks ? tile : tile + (int)gridDim.x, cn = c + 1 < chunks ? c + 1 : 0;
      fresh = tn < tiles;
      if (fresh) {
        load_w(next, tn, cn);
        if (chunks > 1) load_x(xn, cn, xb ^ 1);
      }
      compute(w, x, c, xb);
    }
#pragma unroll
    for (int a = 0; a < NA; ++a) *reinterpret_cast<f32x4*>(&s_acc[buf][wv][a][4 * lane]) = acc[a];
    __syncthreads();  // s_acc[buf] is written again two tiles on, after the next barrier
    if (tid < 256) {
      const int m = (tid >> 2) & 15, nl = 4 * (tid >> 6) + (tid & 3), n = tile * tr + nl;
      if (m < M && nl < tr && n < A.N) {
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < NW; ++i) v[a] += s_acc[buf][i][a][tid];
        A.y[(int64_t)m * A.ys + n] = f2bf(mx_epilogue(A, m, n, v[0], v[1], NA == 2));
      }
    }
  }
}

template <bool XQ, int NA, int SW>
int launch_few_sw(const MxArgs& A, hipStream_t stream) {
  // Tiles that fill the workgroups: as few per workgroup as 16 rows allow, then the rows spread evenly.  Two workgroups
  // to a CU where both fit and have 16 rows each (gated N 7208, K 2304, M 1: 6.9 us, one to a CU 8.1; N 2304: 4.4, 3.7).
  const int wgs = SW <= 3 && A.N > 4096 && (XQ || A.G * A.M * 256 <= 40960) ? 512 : 256;
  const int per = (int)(((int64_t)A.N + 16 * wgs - 1) / (16 * wgs));
  const int tr = (int)(((int64_t)A.N + (int64_t)wgs * per - 1) / ((int64_t)wgs * per));
  const int tiles = (A.N + tr - 1) / tr, grid = (tiles + per - 1) / per;
  int chunks = (A.G + 8 * SW - 1) / (8 * SW), half = 0;
  size_t lds = 0;
  if (!XQ) {
    auto pieces = [&](int c) { return ((A.G + c - 1) / c * A.M * 16 + 511) / 512 * 512; };  // of a chunk's x, whole loads
    if (chunks > 1 || pieces(1) * 16 > kFewLds) {
      if (chunks < 2) chunks = 2;
      while (pieces(chunks) * 32 > kFewLds) ++chunks;
      half = pieces(chunks);
    }
    lds = (size_t)(half ? 2 * half : pieces(1)) * 16;
    if (lds > 16384) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx4_linear_few_kernel<XQ, NA, SW>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return (int)e;
    }
  }
  hipLaunchKernelGGL((mx4_linear_few_kernel<XQ, NA, SW>), dim3(grid), dim3(64 * kFewWaves), lds, stream, A, tr, tiles, chunks,
                     65536 / A.M + 1, half);
  return 0;
}
template <bool XQ, int NA>
int launch_few(const MxArgs& A, hipStream_t stream) {
  if (A.G <= kFewWaves) return launch_few_sw<XQ, NA, 1>(A, stream);
  if (A.G <= 3 * kFewWaves) return launch_few_sw<XQ, NA, 3>(A, stream);
  return launch_few_sw<XQ, NA, XQ && NA == 2 ? 4 : 8>(A, stream);  // (two halves and x: 8 needs more than 256 registers)
}

// ---- more rows: tiles through LDS ----------------------------------------------------------------------------------
// A workgroup of WM x WN waves forms BM rows of x times WN NT 16 rows of W (GATED, NA = 2: every second 16 rows are W2's,
// so a wave holds both sums of an output).  A stage is GS groups of K: x's tile and the scales go straight from memory to
// LDS, one stage ahead.
// W's codes go the same way (loaded in the operands' layout neighbouring lanes lie in different rows, an access to L1 each:
// 4096 a stage of the largest MX4 tile where 512 do, which was its bound), but for the largest bf16 tile, whose x fills LDS:
// there they go to the operand registers, a stage ahead too.  The scales of four groups are loaded at once, 16 bytes a
// row: by single groups their loads were a third of all accesses to L1.
//   bf16: of each group, lane (r, kg) takes row r's block kg, in four products of 32, 8 elements of the block each.
//   MX4: of a stage of two groups, lane (r, kg) takes row r's blocks 2 kg and 2 kg + 1, one in each of two products of
//     128, so that its two scales are one read and the product picks the byte.
// With few tiles K is split over workgroups, whose fp32 sums a second kernel adds in order.
// The outputs go through LDS to 16-byte stores at any alignment, the bias added to the sums once, the residual loaded 64 rows
// ahead (3400 x 24423 of K 248 with both: 142 us; 2-byte accesses at their use 307).
// M 4096, gated N 7208, K 2304: bf16 243 us (1.12 PFLOP/s), MX4 96 (2.8 PFLOP/s).  Neither fills a unit: the matrix cores
// are busy for 49 % and 35 % of the time, LDS for 15 and 23, and the waves are in waits and barriers for 30 % and wait to
// issue for 45 and 34: with two waves to a SIMD a stage's wait, reads, conversions and products run in turn; and 912 tiles
// are 3.6 rounds.  (The clock goes by the inputs' values: of plain normal numbers the same products take 229 and 85 us.)
// M 64, N 32000, K 2304, bf16: 15 us (2.6 TB/s of W; 41 % of the waves' time in waits, one workgroup to a CU and one stage
// ahead).  M 301, N 2304, K 7128, MX4: 13.4 us in 4 splits, and 4.2 for their sums.
constexpr int kGroupM = 4;  // tiles of x that run beside each other for every tile of W (an XCD's L2 holds both)

template <bool XQ, int BM, int WM, int WN, int NT, int NA, int GS, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void mx4_linear_tile_kernel(const MxArgs A, int mtiles, int ntiles, int splits, float* part) {
  constexpr int NB = 2, W = WM * WN, T = 64 * W, MT = BM / (16 * WM), BV = WN * NT * 16, BO = BV / NA;
  constexpr int PR = XQ ? 1 : GS, CH = XQ ? 8 : 16, PL = BM * CH, XL = PR * PL / T;  // planes of a stage, pieces of a row, of a plane
  constexpr bool WLDS = XQ || BM <= 128;                            // W goes through LDS
  constexpr int CW = XQ ? 8 : 4, PW = BV * CW, WL = PR * PW / T;  // as CH, PL, XL for W
  constexpr int XS = BM < 64 ? 64 : BM;
  constexpr int CO = NT / NA * 16;  // a wave's output columns
  static_assert(NT % NA == 0 && PR * PL % T == 0 && PL % 64 == 0 && BV % 64 == 0 && (!WLDS || PR * PW % T == 0) && 4 % GS == 0 && (!XQ || GS == 2), "tile");
  constexpr int EP = W * 16 * (CO + 4) / 4;  // the epilogue's rows
  __shared__ uint4 s_x[NB * PR * PL > EP ? NB * PR * PL : EP];
  __shared__ uint4 s_w[WLDS ? NB : 1][WLDS ? PR * PW : 1], s_ws[2][BV], s_xs[2][XQ ? XS : 1];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kg = lane >> 4, wm = wv / WN, wn = wv % WN, G = A.G;
  // consecutive workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles that share x and W
  int id = blockIdx.x;
  {
    const int all = mtiles * ntiles * splits, per = all / 8, more = all % 8, x = id % 8;
    id = x * per + min(x, more) + id / 8;
  }
  const int split = id % splits;
  id /= splits;
  const int band = id / (kGroupM * ntiles), in = id - band * (kGroupM * ntiles), high = min(kGroupM, mtiles - band * kGroupM);
  const int m0 = (band * kGroupM + in % high) * BM, n0 = in / high * BO;
  const int rows_m = min(BM, A.M - m0), rows_n = min(BO, A.N - n0);
  const int stages = (G + GS - 1) / GS, st0 = (int)((int64_t)stages * split / splits), st1 = (int)((int64_t)stages * (split + 1) / splits);
  const uint32_t wrow = (uint32_t)G * 64, srow = (uint32_t)G * 4;

  const u32x4 rx = XQ ? dma_buf(A.x + (int64_t)m0 * wrow, (uint32_t)rows_m * wrow)
                      : dma_buf(A.x + (int64_t)m0 * A.xs * 2, (uint32_t)(((int64_t)(rows_m - 1) * A.xs + A.K) * 2));
  const u32x4 rxs = dma_buf(XQ ? A.xsc + (int64_t)m0 * srow : A.wsc, XQ ? (uint32_t)rows_m * srow : 0u);
  // (gated: of both halves' rows.  Rows past N give sums that are not stored.)
  const u32x4 rws = dma_buf(A.wsc + (int64_t)n0 * srow, (uint32_t)((NA - 1) * A.N + rows_n) * srow);
  bufrsrc rw[NA];
  u32x4 rwd[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const uint8_t* from = A.W + ((int64_t)a * A.N + n0) * wrow;
    rw[a] = make_buf(from, (uint32_t)rows_n * wrow), rwd[a] = dma_buf(from, (uint32_t)rows_n * wrow);
  }

  // this lane's offsets of a stage's pieces of x: place q of the stage holds piece c of a row
  auto x_piece = [&](int i, int& row, int& gg, int& c) {
    const int q = i * T + tid, p = q % PL;
    gg = q / PL, row = p / CH, c = (p % CH) ^ turn<CH>(row);
  };
  uint32_t vx[XL], vw[WLDS ? WL : NT];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    int row, gg, c;
    x_piece(i, row, gg, c);
    vx[i] = row < rows_m ? (XQ ? (uint32_t)row * wrow : (uint32_t)row * (uint32_t)A.xs * 2) + (uint32_t)(gg * CH + c) * 16 : kOut;
  }
  if constexpr (WLDS) {
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const int q = i * T + tid, p = q % PW, v = p / CW, c = (p % CW) ^ turn<CW>(v);
      vw[i] = (uint32_t)(NA == 2 ? 16 * (v >> 5) + (v & 15) : v) * wrow + (uint32_t)(q / PW * CW + c) * 16;
    }
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) vw[nt] = (uint32_t)(16 * ((wn * NT + nt) / NA) + r) * wrow + 16 * kg;
  }
  auto w_row = [](int v, int N) {  // W's row (from n0) of the tile's row v
    return NA == 2 ? (v >> 4 & 1) * N + 16 * (v >> 5) + (v & 15) : v;
  };
  auto load_stage = [&](int st, int buf) {
    const uint32_t soff = (uint32_t)st * (PR * CH * 16);
    const bool tail = XQ ? (st + 1) * GS > G : (st + 1) * GS * 128 > A.K;  // uniform: the row ends within the stage
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      uint32_t v = vx[i];
      if (tail) {
        int row, gg, c;
        x_piece(i, row, gg, c);
        if (XQ ? st * GS + (c >> 2) >= G : 128 * (st * GS + gg) + 8 * c >= A.K) v = kOut;
      }
      dma16(rx, lds_address(&s_x[buf * PR * PL + i * T + 64 * wv]), v, soff);
    }
    if constexpr (WLDS) {
      // a wave's 64 pieces are rows of one half.  (A group past the row's end is of the next row, or 0; x's is 0.)
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        u32x4 from = rwd[0];
        if constexpr (NA == 2) {
          const bool second = (i * T + 64 * wv) % PW / CW >> 4 & 1;
          from.x = __builtin_amdgcn_readfirstlane(second ? rwd[1].x : rwd[0].x);
          from.y = __builtin_amdgcn_readfirstlane(second ? rwd[1].y : rwd[0].y);
        }
        dma16(from, lds_address(&s_w[WLDS ? buf : 0][i * T + 64 * wv]), vw[i], (uint32_t)st * (64 * GS));
      }
    }
  };
  auto load_scales = [&](int four) {  // of groups 4 four to 4 four + 3 (past the row's end: of the next row, not used or masked)
#pragma unroll
    for (int i = wv; i < BV / 64; i += W)
      dma16(rws, lds_address(&s_ws[four & 1][i * 64]), (uint32_t)w_row(i * 64 + lane, A.N) * srow, (uint32_t)four * 16);
    if constexpr (XQ)
#pragma unroll
      for (int i = wv; i < XS / 64; i += W)
        dma16(rxs, lds_address(&s_xs[four & 1][i * 64]), i * 64 + lane < rows_m ? (uint32_t)(i * 64 + lane) * srow : kOut, (uint32_t)four * 16);
  };
  // (a group past the row's end is of the next row, or 0; x's is 0)
  auto load_w = [&](uint4 (*c)[NT], int st) {
#pragma unroll
    for (int gg = 0; gg < GS; ++gg)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        c[gg][nt] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(rw[(wn * NT + nt) % NA], vw[nt] + 64 * gg, (uint32_t)st * (64 * GS), 0));
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Stage st + 1 is issued when st begins, into the buffer that st - 1 has left.  (Two or three stages ahead, or the groups
  // of a stage shared between twice the waves, took the same time: M 32, gated N 7208, K 2304, bf16 11.9, 11.8 and 12.1 us.)
  uint4 w[GS][NT], next[GS][NT];
  auto issue = [&](int st) {
    if constexpr (!WLDS) load_w(next, st);
    if (st == st0 || (st * GS & 3) == 0) load_scales(st * GS >> 2);
    load_stage(st, (st - st0) % NB);
  };
  if (st0 < st1) issue(st0);
  for (int st = st0; st < st1; ++st) {
    const int buf = (st - st0) % NB;
    dma_wait();  // this wave's part of the stage has come,
    __syncthreads();  // everybody's has, and the buffer of the stage before has been read
    if constexpr (!WLDS)
#pragma unroll
      for (int q = 0; q < GS * NT; ++q) {
        const int gg = q / NT, nt = q % NT;
        w[gg][nt] = next[gg][nt];
        asm volatile("" : "+v"(w[gg][nt].x), "+v"(w[gg][nt].y), "+v"(w[gg][nt].z), "+v"(w[gg][nt].w));
      }
    if (st + 1 < st1) issue(st + 1);
    if constexpr (XQ) {
      // the scales of blocks 2 kg and 2 kg + 1, in bytes 0 and 1 (a group past the row's end: 0)
      const uint32_t keep = 2 * st + 1 >= G && kg >= 2 ? 0u : 0xffffu;
      const int sb = st >> 1 & 1, so = (st & 1) * 4 + kg;
      uint32_t ws[NT];
      i32x8 wf[2][NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        ws[nt] = reinterpret_cast<const uint16_t*>(s_ws[sb])[((wn * NT + nt) * 16 + r) * 8 + so] & keep;
        const uint4* row = s_w[WLDS ? buf : 0] + ((wn * NT + nt) * 16 + r) * CW;
        wf[0][nt] = codes8(row[(2 * kg) ^ turn<CW>(r)]), wf[1][nt] = codes8(row[(2 * kg + 1) ^ turn<CW>(r)]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int row = (wm * MT + mt) * 16 + r;
        const uint32_t xs = reinterpret_cast<const uint16_t*>(s_xs[sb])[row * 8 + so] & keep;
        const i32x8 x0 = codes8(s_x[buf * PR * PL + row * CH + ((2 * kg) ^ turn<CH>(r))]);
        const i32x8 x1 = codes8(s_x[buf * PR * PL + row * CH + ((2 * kg + 1) ^ turn<CH>(r))]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][mt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[0][nt], x0, acc[nt][mt], 4, 4, 0, ws[nt], 0, xs);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][mt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[1][nt], x1, acc[nt][mt], 4, 4, 1, ws[nt], 1, xs);
      }
    } else {
#pragma unroll
      for (int gg = 0; gg < GS; ++gg) {
        if (GS > 1 && GS * st + gg >= G) break;  // uniform
        const int g = GS * st + gg;
        uint32_t ws[NT];
        uint4 wc[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int v = (wn * NT + nt) * 16 + r;
          ws[nt] = reinterpret_cast<const uint8_t*>(s_ws[g >> 2 & 1])[v * 16 + (g & 3) * 4 + kg];
          wc[nt] = WLDS ? s_w[WLDS ? buf : 0][gg * PW + v * CW + (kg ^ turn<CW>(r))] : w[gg][nt];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 wf[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t c = j == 0 ? wc[nt].x : j == 1 ? wc[nt].y : j == 2 ? wc[nt].z : wc[nt].w;
            wf[nt] = deq8(c, __uint_as_float(ws[nt] << 23));
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int row = (wm * MT + mt) * 16 + r;
            const uint4 xf = s_x[buf * PR * PL + gg * PL + row * CH + ((4 * kg + j) ^ turn<CH>(r))];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[nt][mt] = mfma(wf[nt], xf, acc[nt][mt]);
          }
        }
      }
    }
  }

  if constexpr (SPLIT) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + (wm * MT + mt) * 16 + r, n = n0 + 16 * ((wn * NT + nt) / NA) + 4 * kg;
        if (m >= A.M || n >= A.N) continue;
        float* p = part + (((int64_t)split * A.M + m) * NA + (nt % NA)) * A.N + n;
        if ((A.N & 3) == 0) {
          *reinterpret_cast<f32x4*>(p) = acc[nt][mt];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < A.N) p[i] = acc[nt][mt][i];
        }
      }
  } else {
    // 16 rows of the wave at a time through LDS (each wave's own part of x's buffers), so that a lane stores 8 columns;
    // the residual of the next kAhead of them is on its way meanwhile
    constexpr int LD = CO + 4;  // floats: rows start 4 banks apart
    constexpr int EI = (16 * CO / 8 + 63) / 64, kAhead = MT < 4 ? MT : 4;
    float* own = reinterpret_cast<float*>(s_x) + wv * 16 * LD;
    uint4 rv[kAhead][EI];
    auto load_res = [&](int mt) {
#pragma unroll
      for (int i = 0; i < EI; ++i) {
        const int e = i * 64 + lane, m = m0 + (wm * MT + mt) * 16 + e / (CO / 8), n = n0 + wn * CO + e % (CO / 8) * 8;
        if (e < 16 * CO / 8 && m < A.M && n + 8 <= A.N) rv[mt % kAhead][i] = load16(A.res + (int64_t)m * A.rs + n);
      }
    };
    if (A.bias)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int n = n0 + 16 * ((wn * NT + nt) / NA) + 4 * kg;
        const bf16_t* b = A.bias + nt % NA * (int64_t)A.N + n;
        f32x4 add;
#pragma unroll
        for (int i = 0; i < 4; ++i) add[i] = n + i < A.N ? bf2f(b[i]) : 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[nt][mt] += add;
      }
    if (A.res)
#pragma unroll
      for (int mt = 0; mt < kAhead; ++mt) load_res(mt);
    __syncthreads();  // x's last stage has been read
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; nt += NA) {
        f32x4 v = acc[nt][mt], v2 = acc[nt + NA - 1][mt];
        if constexpr (NA == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = mx_gate(v[i], v2[i]);
        }
        *reinterpret_cast<f32x4*>(own + r * LD + 16 * (nt / NA) + 4 * kg) = v;
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < EI; ++i) {
        const int e = i * 64 + lane, row = e / (CO / 8), col = e % (CO / 8) * 8;
        const int m = m0 + (wm * MT + mt) * 16 + row, n = n0 + wn * CO + col;
        if (e >= 16 * CO / 8 || m >= A.M || n >= A.N) continue;
        float v[8];
        *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(own + row * LD + col);
        *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(own + row * LD + col + 4);
        const bf16_t* res = A.res ? A.res + (int64_t)m * A.rs + n : nullptr;
        bf16_t* y = A.y + (int64_t)m * A.ys + n;
        if (n + 8 <= A.N) {
          if (res) {
            const uint4 u = rv[mt % kAhead][i];
            const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) v[2 * q] += __uint_as_float(h[q] << 16), v[2 * q + 1] += __uint_as_float(h[q] & 0xffff0000u);
          }
          uint32_t h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = (uint32_t)f2bf(v[2 * q]) | ((uint32_t)f2bf(v[2 * q + 1]) << 16);
          store16(y, uint4{h[0], h[1], h[2], h[3]});
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (n + q < A.N) y[q] = f2bf(v[q] + (res ? bf2f(res[q]) : 0.f));
        }
      }
      if (A.res && mt + kAhead < MT) load_res(mt + kAhead);
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// y = epilogue(the splits' sums, added in order), four columns per thread (V 4: N % 4 == 0) or one.  Four splits' sums are
// loaded at once (one after the other, M 32, N 2304, 12 splits: 6.2 us, now 4.6).
template <int NA, int V>
__global__ __launch_bounds__(256) void mx4_linear_sum_kernel(const MxArgs A, const float* part, int splits) {
  constexpr int U = 4;
  const int n = (blockIdx.x * 256 + threadIdx.x) * V, m = blockIdx.y;
  if (n >= A.N) return;
  const int64_t step = (int64_t)A.M * NA * A.N;  // from a split to the next
  const float* p = part + (int64_t)m * NA * A.N + n;
  float v[NA][V] = {};
  for (int s = 0; s < splits; s += U) {
    float f[U][NA][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        const float* q = p + min(s + u, splits - 1) * step + (int64_t)a * A.N;
        if constexpr (V == 4)
          *reinterpret_cast<f32x4*>(f[u][a]) = *reinterpret_cast<const f32x4*>(q);
        else
          f[u][a][0] = *q;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int i = 0; i < V; ++i) v[a][i] += s + u < splits ? f[u][a][i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) A.y[(int64_t)m * A.ys + n + i] = f2bf(mx_epilogue(A, m, n + i, v[0][i], v[NA - 1][i], NA == 2));
}

// The tile and the split of K of a product: the least estimated time, rounds of 256 workgroups (one to a CU) of so many
// groups each.  The times per group, and those of a split (its sums written, and added by another kernel), were fitted to 344
// measured products (M 32 to 4096, N 2304 to 32000, K 2304 and 7208, every tile, splits 1 to 8): the estimate is within
// a tenth of most of them, and the tile it takes within a tenth of the best.
struct MxTile {
  int bm, bv;
  float bf16, mx4;  // us per group of 128
};
constexpr MxTile kTiles[5] = {
    {32, 128, 0.36f, 0.24f}, {64, 128, 0.60f, 0.27f}, {128, 128, 0.97f, 0.37f}, {128, 256, 1.57f, 0.66f}, {256, 256, 3.13f, 1.14f}};
struct MxPlan {
  int kind, bo, mtiles, ntiles, splits;  // kind 0: the kernel for few rows, otherwise kTiles[kind - 1]
  size_t bytes;
  MxPlan(int M, int N, int K, bool xq, bool gated) {
    const int NA = gated ? 2 : 1, G = (int)(((int64_t)K + 127) / 128);
    kind = bo = mtiles = ntiles = splits = 0, bytes = 0;
    // (N 32000, K 2304, M 16: 18.0 us by the kernel for few rows, 11.5 in tiles; N 2 x 7208: 8.4 and 10.7)
    if (M <= 16 && (int64_t)N * NA < 20000) return;
    float best = 0.f;
    for (int k = 0; k < 5; ++k) {
      const MxTile& t = kTiles[k];
      const int mt = (M + t.bm - 1) / t.bm, nt = (int)(((int64_t)N * NA + t.bv - 1) / t.bv);
      const int64_t all = (int64_t)mt * nt;
      for (int s = 1; s <= 16 && (s == 1 || (M > 16 && s <= G / 4 && all * s <= 512)); ++s) {
        float us = (float)((all * s + 255) / 256) * (float)((G + s - 1) / s) * (xq ? t.mx4 : t.bf16);
        if (s > 1) us += 3.5f + (float)s * M * N * NA * 8.f / 5e6f;
        if (kind == 0 || us < best) best = us, kind = k + 1, mtiles = mt, ntiles = nt, splits = s, bo = t.bv / NA;
      }
    }
    if (splits > 1) bytes = (size_t)splits * M * N * NA * 4;
  }
};

template <bool XQ, int BM, int WM, int WN, int NT, int NA, int GS>
void launch_tile(const MxArgs& A, const MxPlan& P, float* part, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)P.mtiles * P.ntiles * P.splits)), block(64 * WM * WN);
  if (P.splits > 1) {
    hipLaunchKernelGGL((mx4_linear_tile_kernel<XQ, BM, WM, WN, NT, NA, GS, true>), grid, block, 0, stream, A, P.mtiles, P.ntiles, P.splits, part);
    if (A.N % 4 == 0)
      hipLaunchKernelGGL((mx4_linear_sum_kernel<NA, 4>), dim3((A.N / 4 + 255) / 256, A.M), dim3(256), 0, stream, A, part, P.splits);
    else
      hipLaunchKernelGGL((mx4_linear_sum_kernel<NA, 1>), dim3((A.N + 255) / 256, A.M), dim3(256), 0, stream, A, part, P.splits);
  } else {
    hipLaunchKernelGGL((mx4_linear_tile_kernel<XQ, BM, WM, WN, NT, NA, GS, false>), grid, block, 0, stream, A, P.mtiles, P.ntiles, 1, part);
  }
}

template <bool XQ, int NA>
int launch_linear(const MxArgs& A, const MxPlan& P, float* part, hipStream_t stream) {
  if (P.kind == 0) return launch_few<XQ, NA>(A, stream);
  if (P.kind == 1)
    launch_tile<XQ, 32, 1, 4, 2, NA, 2>(A, P, part, stream);
  else if (P.kind == 2)
    launch_tile<XQ, 64, 2, 4, 2, NA, 2>(A, P, part, stream);
  else if (P.kind == 3)
    launch_tile<XQ, 128, 2, 4, 2, NA, XQ ? 2 : 1>(A, P, part, stream);
  else if (P.kind == 4)
    launch_tile<XQ, 128, 2, 4, 4, NA, XQ ? 2 : 1>(A, P, part, stream);
  else
    launch_tile<XQ, 256, 2, 4, 4, NA, XQ ? 2 : 1>(A, P, part, stream);
  return 0;
}

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

extern "C" int kdn_mx4_quantize(const void* x, int x_bf16, int64_t x_row_stride, int64_t rows, int cols, void* codes,
                                void* scales, hipStream_t stream) {
  if (rows < 0 || cols < 1 || (rows > 1 && x_row_stride < cols) || (x_bf16 != 0 && x_bf16 != 1)) return KDN_ERR_ARG;
  if (rows == 0) return 0;
  if (!x || !codes || !scales || !aligned(codes, 16) || !aligned(scales, 4) || !aligned(x, x_bf16 ? 2 : 4)) return KDN_ERR_ARG;
  const int64_t G = ((int64_t)cols + 127) / 128, per = 16 * G;
  const int64_t slab = (1ll << 30) / per > 0 ? (1ll << 30) / per : 1;  // 32-bit item counts
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = rows - r0 < slab ? rows - r0 : slab, items = n * per;
    const dim3 grid((unsigned)((items + 255) / 256));
    uint32_t* c = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(codes) + r0 * 64 * G);
    uint8_t* s = static_cast<uint8_t*>(scales) + r0 * 4 * G;
    if (x_bf16)
      hipLaunchKernelGGL(mx4_quantize_kernel<bf16_t>, grid, dim3(256), 0, stream, static_cast<const bf16_t*>(x) + r0 * x_row_stride,
                         x_row_stride, cols, (uint32_t)per, (uint32_t)items, c, s);
    else
      hipLaunchKernelGGL(mx4_quantize_kernel<float>, grid, dim3(256), 0, stream, static_cast<const float*>(x) + r0 * x_row_stride,
                         x_row_stride, cols, (uint32_t)per, (uint32_t)items, c, s);
  }
  KDN_CHECK_LAUNCH();
  return 0;
}

extern "C" int kdn_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int cols, void* y, int y_bf16,
                                  hipStream_t stream) {
  if (rows < 0 || cols < 1 || (y_bf16 != 0 && y_bf16 != 1)) return KDN_ERR_ARG;
  if (rows == 0) return 0;
  if (!y || !codes || !scales || !aligned(codes, 16) || !aligned(scales, 4) || !aligned(y, y_bf16 ? 2 : 4)) return KDN_ERR_ARG;
  const int64_t G = ((int64_t)cols + 127) / 128, per = (y_bf16 ? 16 : 32) * G;
  const int64_t slab = (1ll << 30) / per > 0 ? (1ll << 30) / per : 1;
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = rows - r0 < slab ? rows - r0 : slab, items = n * per;
    const dim3 grid((unsigned)((items + 255) / 256));
    const uint8_t* c = static_cast<const uint8_t*>(codes) + r0 * 64 * G;
    const uint8_t* s = static_cast<const uint8_t*>(scales) + r0 * 4 * G;
    if (y_bf16)
      hipLaunchKernelGGL(mx4_dequantize_kernel<bf16_t>, grid, dim3(256), 0, stream, c, s, cols, (uint32_t)per, (uint32_t)items,
                         static_cast<bf16_t*>(y) + r0 * cols);
    else
      hipLaunchKernelGGL(mx4_dequantize_kernel<float>, grid, dim3(256), 0, stream, c, s, cols, (uint32_t)per, (uint32_t)items,
                         static_cast<float*>(y) + r0 * cols);
  }
  KDN_CHECK_LAUNCH();
  return 0;
}

extern "C" size_t kdn_mx4_linear_workspace_size(int M, int N, int K, int x_mx4, int gated) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return MxPlan(M, N, K, x_mx4 != 0, gated != 0).bytes;
}

extern "C" int kdn_mx4_linear(const void* x, const void* x_scales, int64_t x_row_stride, const void* W, const void* W_scales,
                              const void* bias, const void* res, int64_t res_row_stride, int M, int N, int K, int gated,
                              void* y, int64_t y_row_stride, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || N < 0 || K < 1 || (gated != 0 && gated != 1)) return KDN_ERR_ARG;
  if (M == 0 || N == 0) return 0;
  const bool xq = x_scales != nullptr;
  if (!x || !W || !W_scales || !y || !aligned(x, 16) || !aligned(W, 16) || !aligned(W_scales, 4) || !aligned(x_scales, 4) ||
      !aligned(y, 2) || !aligned(bias, 2) || !aligned(res, 2) || (M > 1 && y_row_stride < N) || (res && M > 1 && res_row_stride < N))
    return KDN_ERR_ARG;
  if (!xq && (K % 8 || (M > 1 && (x_row_stride < K || x_row_stride % 8)))) return KDN_ERR_ARG;
  // a tile's rows are addressed by 32-bit offsets
  if (K > (1 << 20) || (int64_t)N * K >= (1ll << 34) || (!xq && M > 1 && x_row_stride > (1 << 21))) return KDN_ERR_ARG;
  const MxPlan P(M, N, K, xq, gated != 0);
  if (P.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < P.bytes)) return KDN_ERR_ARG;
  if ((int64_t)P.mtiles * P.ntiles * P.splits > 0x7fffffffll || (P.splits > 1 && M > 65535)) return KDN_ERR_ARG;
  const int G = (int)(((int64_t)K + 127) / 128);
  const MxArgs A{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(x_scales), M > 1 ? x_row_stride : K,
                 static_cast<const uint8_t*>(W), static_cast<const uint8_t*>(W_scales), static_cast<const bf16_t*>(bias),
                 static_cast<const bf16_t*>(res), res_row_stride, M, N, K, G, static_cast<bf16_t*>(y), y_row_stride};
  float* part = static_cast<float*>(workspace);
  const int e = xq ? (gated ? launch_linear<true, 2>(A, P, part, stream) : launch_linear<true, 1>(A, P, part, stream))
                   : (gated ? launch_linear<false, 2>(A, P, part, stream) : launch_linear<false, 1>(A, P, part, stream));
  if (e != 0) return e;
  KDN_CHECK_LAUNCH();
  return 0;
}
