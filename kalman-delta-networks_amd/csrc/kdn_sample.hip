// One token per row of logits: temperature, top-k, top-p and min-p, and a draw from given exponential noise.
// The reference has no counterpart (it trains and evaluates on whole sequences).
//
// With p_i = exp((l_i - max l) / T), the tokens are ordered by (l descending, index ascending); top-k keeps the first
// k, top-p of these the shortest prefix whose mass reaches top_p of theirs, min-p those with p_i >= min_p.  For noise
// e_i ~ Exp(1), argmax p_i / e_i over the kept is distributed as p restricted to them: each e_i / p_i is exponential
// with rate p_i, and the smallest of such is i with probability p_i / sum p.
//
// The order of a row is never formed.  The keys (l's bits made monotone, then the index from behind) are distinct, so
// a truncation is a threshold on the key:
//   * few candidates.  Of the 1024 threads' largest logits the k-th is at most the k-th of the row, so for k up to 192
//     all tokens above that bound (about k of them) go to a list in LDS and are ranked there, each with the mass before it:
//     top-k, top-p, min-p and the draw then look at the list alone.
//   * otherwise a radix selection: a histogram, over the keys still in question, of their count (top-k) or mass (top-p);
//     the digit where the count reaches k, or the mass top_p of the whole, holds the threshold, and its keys, when they
//     fit the list, are ranked there.  The first digit is (max l - l) / T in 32nds of a factor of two, which spreads the
//     likely tokens over its 2048 values, so the list mostly follows at once; otherwise (`refine`) the digits go on below
//     the highest bit in which the keys in question differ.  A token of p below (1 - top_p) / V of the mass can not be in
//     the prefix (all such tokens together hold less than 1 - top_p) and is left out of the mass histogram.
// Masses are whole multiples of 2^-40 of the largest p, so their sums do not depend on the order of the atomic
// additions and a row's token is the same in every run (2^20 such masses fit 64 bits).
//
// One workgroup per row; the row is read from memory once, in 16-byte pieces that stay in LDS (of a longer row the rest
// is read again from L2 by every pass).  Noise is read for the pieces that hold a kept token.  Bound by the passes
// over the row on its one CU, one after the other (each operation on all of 32000 tokens is 500 cycles of its vector ALU): with
// settings of their own 64 rows of 32000 take 26 us, in which the ALUs of their 64 CUs issue for 43 % of the time, the waves
// spend 60 % in waits (barriers, LDS atomics, loads), and the other CUs are idle.  256 rows of 50304 fp32 with top-p and
// min-p: 39 us, 41 % and 67 % (the first pass and the draw wait for HBM).  bf16, one row of 32000: top-k 50 and top-p 9.0 us,
// nothing 9.6, top-p alone 16, greedy 7.3.
#include "kdn_common.h"
#include "../../include/kdn.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kList = 256;
// Candidates are listed for k up to this: 64 rows of 32000 bf16 with top-p take 10.2 us for k 50, 13.6 for 150 and 16.1 for
// 200 (by selection 20.9, 21.5 and 22.0); of k 250 there are more than the list holds, and 26.8 us (by selection 22.1).
constexpr int kFew = 192;
constexpr int kIdxBits = 20;
constexpr float kMassOne = 1099511627776.f;  // 2^40

typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t ls;
  const float* noise;
  int64_t ns;
  const float* tv;
  float t;
  const int* kv;
  int k;
  const float* pv;
  float p;
  const float* mv;
  float m;
  int V;
  int pieces, resident;  // see Row
  int64_t* tokens;
  float* logprobs;
};

struct Half {
  uint16_t u;
};
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float get(uint4 v, int e) { return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w); }
};
template <> struct Elem<bf16_t> {
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ float get(uint4 v, int e) {
    const uint32_t w = e / 2 == 0 ? v.x : e / 2 == 1 ? v.y : e / 2 == 2 ? v.z : v.w;
    return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <> struct Elem<Half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ float get(uint4 v, int e) {
    const uint32_t w = e / 2 == 0 ? v.x : e / 2 == 1 ? v.y : e / 2 == 2 ? v.z : v.w;
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w >> 16 : w));
  }
};

// l's bits as an unsigned number of the same order (-0 as 0, so that equal logits have equal keys)
__device__ __forceinline__ uint32_t ordered(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ u64 key_of(float l, int i) {
  return ((u64)ordered(l) << kIdxBits) | (uint32_t)((1 << kIdxBits) - 1 - i);
}
__device__ __forceinline__ float key_logit(u64 key) {
  const uint32_t o = (uint32_t)(key >> kIdxBits);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int key_index(u64 key) { return (1 << kIdxBits) - 1 - (int)(key & ((1u << kIdxBits) - 1)); }

struct Shared {
  uint32_t cnt[kBins];
  u64 w[kBins];
  u64 list[kList], listw[kList], run[kList];
  uint32_t rank[kList];
  float redf[3][kWaves];
  u64 redw[2][kWaves];
  uint32_t n;
  int flag, index;
  // the selection's answer: the digit, and the count (or mass) of the digits before it; the threshold's key
  int digit;
  u64 before;
  u64 key;
};

// ---- reductions ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float max_raw(float a, float b) {  // one instruction; NaN is dealt with apart
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {
  return max_raw(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float row16_max(float x) {
  return dpp_max<kDppMirror>(dpp_max<kDppHalfMirror>(dpp_max<kDppXor2>(dpp_max<kDppXor1>(x))));
}
// over the workgroup: sums in a fixed order / maxima; `slot` separates calls that no barrier lies between
__device__ __forceinline__ float block_add(Shared& S, int slot, float v) {
  v = swz16_add(row16_sum(v));
  v += __shfl_xor(v, 32, 64);
  if ((threadIdx.x & 63) == 0) S.redf[slot][threadIdx.x >> 6] = v;
  __syncthreads();
  return row16_sum(S.redf[slot][threadIdx.x & 15]);
}
__device__ __forceinline__ float block_max(Shared& S, int slot, float v) {
  v = row16_max(v);
  v = max_raw(v, __shfl_xor(v, 16, 64));
  v = max_raw(v, __shfl_xor(v, 32, 64));
  if ((threadIdx.x & 63) == 0) S.redf[slot][threadIdx.x >> 6] = v;
  __syncthreads();
  return row16_max(S.redf[slot][threadIdx.x & 15]);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_u64(u64 v) {  // 0 where the lane has no source, or is not in ROWS
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
  return ((u64)(uint32_t)hi << 32) | (uint32_t)lo;
}
__device__ __forceinline__ u64 row16_scan(u64 v) {  // inclusive, within rows of 16 lanes (row_shr 1, 2, 4, 8)
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {  // inclusive (then row_bcast 15 and 31)
  v = row16_scan(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 read_lane(u64 v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane);
  return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 block_add(Shared& S, u64 v) {
  v = wave_scan(v);
  if ((threadIdx.x & 63) == 63) S.redw[1][threadIdx.x >> 6] = v;
  __syncthreads();
  return read_lane(row16_scan(S.redw[1][threadIdx.x & 15]), 15);
}

// The first digit (0, 1, ...) at which base and the running sum of `h` reach `want`: S.digit (-1: none), S.before.
template <typename H>
__device__ __forceinline__ void pick_digit(Shared& S, const H* h, u64 base, u64 want) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const u64 a = h[2 * tid], b = h[2 * tid + 1], sum = wave_scan(a + b);
  if (lane == 63) S.redw[0][wv] = sum;
  if (tid == 0) S.digit = -1;
  __syncthreads();
  const u64 waves = row16_scan(S.redw[0][lane & 15]);
  const u64 run = base + sum - a - b + (wv ? read_lane(waves, wv - 1) : 0ull);
  if (run < want && run + a >= want) S.digit = 2 * tid, S.before = run;
  if (run + a < want && run + a + b >= want) S.digit = 2 * tid + 1, S.before = run + a;
  __syncthreads();
}

// ---- a token's place in the distribution ------------------------------------------------------------------------
struct Dist {
  float mx, ct, t;  // the largest logit, log2(e) / T, T
  __device__ __forceinline__ float log2p(float x) const { return (x - mx) * ct; }
  __device__ __forceinline__ float z(float x) const { return x == mx ? 0.f : (x - mx) / t; }
  __device__ __forceinline__ float prob(float x) const { return expf(z(x)); }
};
__device__ __forceinline__ int first_digit(float y) { return (int)fminf(y * -32.f, (float)(kBins - 1)); }
// p <= 1 in 2^-40ths: the low bits of p + 2^12 in double precision, whose last place that is
__device__ __forceinline__ u64 mass_of(float p) {
  return (u64)__double_as_longlong((double)p + 4096.0) - 0x40b0000000000000ull;
}
// token i of logit x is not behind (thr_x, thr_i)
__device__ __forceinline__ bool stays(float x, int i, float thr_x, int thr_i) {
  return x > thr_x || (x == thr_x && i <= thr_i);
}

// The row in pieces of 16 bytes, piece `it` of a thread at (it kThreads + tid): the first kThreads * resident of them are
// kept in LDS, the others read from L2 in every pass.  The passes are rolled loops over the pieces: with the row in
// registers, every pass unrolled over them, the code was 60 to 70 KB, past the instruction cache.
constexpr int kResident = 8;  // 16 KB each
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* l;
  uint4* kept;
  int V, pieces, resident;  // pieces: per thread
  bool odd;                 // the row holds NaN, or its largest logit `top` is +inf: see tidy()
  float top;

  static __device__ __forceinline__ float element(const T* p, int i) {
    uint4 v = uint4{0u, 0u, 0u, 0u};
    if constexpr (sizeof(T) == 4)
      v.x = __float_as_uint(reinterpret_cast<const float*>(p)[i]);
    else
      v.x = reinterpret_cast<const uint16_t*>(p)[i];
    return Elem<T>::get(v, 0);
  }
  // NaN cannot be drawn (-inf); if the largest logit is +inf, it alone can: 0 there, -inf elsewhere
  __device__ __forceinline__ float tidy(float x) const {
    if (!(x > -INFINITY)) return -INFINITY;
    return top < INFINITY ? x : (x < top ? -INFINITY : 0.f);
  }
  __device__ __forceinline__ float logit(int i) const {
    const float x = element(l, i);
    return odd ? tidy(x) : x;
  }
  __device__ __forceinline__ uint4 fetch(int it) const {  // -inf past the row's end
    const int i = (it * kThreads + (int)threadIdx.x) * E;
    if (i + E <= V) return load16(l + i);
    uint32_t w[4] = {Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf};
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (i + e < V) {
        if constexpr (sizeof(T) == 4) {
          w[e] = __float_as_uint(reinterpret_cast<const float*>(l)[i + e]);
        } else {
          const uint32_t u = reinterpret_cast<const uint16_t*>(l)[i + e];
          w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | (u << 16) : (w[e / 2] & 0xffff0000u) | u;
        }
      }
    return uint4{w[0], w[1], w[2], w[3]};
  }
  __device__ __forceinline__ void unpack(uint4 c, float* x) const {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = Elem<T>::get(c, e);
    if (odd) {  // uniform, rare
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = tidy(x[e]);
    }
  }
  __device__ __forceinline__ uint4 piece(int it) const {
    return it < resident ? kept[it * kThreads + threadIdx.x] : fetch(it);
  }
  // fn(x, i): a piece's logits and its first one's index
  template <typename F>
  __device__ __forceinline__ void each(F&& fn) const {
#pragma unroll 1
    for (int it = 0; it < pieces; ++it) {
      float x[E];
      unpack(piece(it), x);
      fn(x, (it * kThreads + (int)threadIdx.x) * E);
    }
  }
};

// S.run[i] = the sum of listw (S.rank[i] = the number) of the n <= kList listed keys above key i.  Every wave takes a
// 16th of the keys to compare with (one thread comparing with all 60 to 200 of them took 2 us).
__device__ __forceinline__ void rank_list(Shared& S, int n) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  if (tid < n) S.run[tid] = 0, S.rank[tid] = 0;
  __syncthreads();
  for (int i = lane; i < n; i += 64) {
    const u64 mine = S.list[i];
    u64 run = 0;
    uint32_t rank = 0;
#pragma unroll 2
    for (int j = wv; j < n; j += kWaves) {
      const bool first = S.list[j] > mine;
      rank += first, run += first ? S.listw[j] : 0ull;
    }
    if (rank) atomicAdd(&S.rank[i], rank), atomicAdd(&S.run[i], run);
  }
  __syncthreads();
}
// The listed key at which `before` and the running sum reach `want`: S.key (false: more keys than the list holds)
__device__ __forceinline__ bool pick_key(Shared& S, int n, u64 before, u64 want) {
  if (n > kList) return false;
  rank_list(S, n);
  const int tid = threadIdx.x;
  if (tid < n) {
    const u64 run = before + S.run[tid];
    if (run < want && run + S.listw[tid] >= want) S.key = S.list[tid];
  }
  __syncthreads();
  return true;
}

// The selection where more keys share the first digit b than the list holds (ties, or a temperature that gathers the
// row in few digits): by further digits, over the row in memory.  -> S.key.
template <bool MASS, typename R>
__device__ __forceinline__ void refine(Shared& S, const R& row, const Dist& D, int b, u64 before, u64 want, float thr_x, int thr_i) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  int shift = 32 + kIdxBits;
  u64 prefix = 0;
  auto each = [&](auto&& fn) {
#pragma unroll 1
    for (int i = tid; i < row.V; i += kThreads) {
      const float x = row.logit(i), y = D.log2p(x);
      const u64 key = key_of(x, i);
      if (x > -INFINITY && first_digit(y) == b && stays(x, i, thr_x, thr_i) && (key >> shift) == prefix)
        fn(key, MASS ? mass_of(fexp2(y)) : 1ull);
    }
  };
  while (true) {
    // the highest bit in which the keys differ (they are distinct: there is one)
    u64 lo = ~0ull, hi = 0;
    each([&](u64 key, u64) { lo = key < lo ? key : lo, hi = key > hi ? key : hi; });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const u64 a = __shfl_xor(lo, o, 64), c = __shfl_xor(hi, o, 64);
      lo = a < lo ? a : lo, hi = c > hi ? c : hi;
    }
    if (lane == 0) S.redw[0][wv] = lo, S.redw[1][wv] = hi;
    for (int i = tid; i < kBins; i += kThreads) S.w[i] = 0;
    if (tid == 0) S.n = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < kWaves; ++i)
      lo = S.redw[0][i] < lo ? S.redw[0][i] : lo, hi = S.redw[1][i] > hi ? S.redw[1][i] : hi;
    __syncthreads();  // redw is written again by pick_digit
    const int upto = lo < hi ? 64 - __clzll((long long)(lo ^ hi)) : 1;
    const int next = upto > 11 ? upto - 11 : 0, last = (1 << (upto - next)) - 1;
    // descending keys: ascending digits
    each([&](u64 key, u64 w) { atomicAdd(&S.w[last - (int)((key >> next) & (u64)last)], w); });
    __syncthreads();
    pick_digit(S, S.w, before, want);
    if (S.digit < 0) return;  // cannot be: the sums reach `want`
    before = S.before;
    prefix = ((hi >> upto) << (upto - next)) | (u64)(last - S.digit), shift = next;
    each([&](u64 key, u64 w) {
      const uint32_t at = atomicAdd(&S.n, 1u);
      if (at < (uint32_t)kList) S.list[at] = key, S.listw[at] = w;
    });
    __syncthreads();
    if (pick_key(S, (int)S.n, before, want)) return;
    __syncthreads();
  }
}

// The token at which, in descending order, the count (MASS: the mass) of those that stay above (thr_x, thr_i) reaches
// `want`, its first digit and the sum before that being S.digit, S.before: (thr_x, thr_i).  Whether the list sufficed
// (S.list, S.n hold the digit's keys then, and S.w is as it was).
template <bool MASS, typename R>
__device__ __forceinline__ bool select_key(Shared& S, const R& row, const Dist& D, u64 want, float& thr_x, int& thr_i) {
  const int b = S.digit;
  const u64 before = S.before;
  if (threadIdx.x == 0) S.n = 0, S.key = ~0ull;
  __syncthreads();
  // first_digit(y) == b (scaling by 32 is exact), and not -inf
  const float hi = (float)b * (-1.f / 32.f), lo = b == kBins - 1 ? -INFINITY : (float)(b + 1) * (-1.f / 32.f);
  row.each([&](const float* x, int i) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < R::E; ++e) {
      const float y = D.log2p(x[e]);
      any |= y <= hi && y > lo;
    }
    if (!any) return;
#pragma unroll
    for (int e = 0; e < R::E; ++e) {
      const float y = D.log2p(x[e]);
      if (y <= hi && y > lo && stays(x[e], i + e, thr_x, thr_i)) {
        const uint32_t at = atomicAdd(&S.n, 1u);
        if (at < (uint32_t)kList) S.list[at] = key_of(x[e], i + e), S.listw[at] = MASS ? mass_of(fexp2(y)) : 1;
      }
    }
  });
  __syncthreads();
  const bool ranked = pick_key(S, (int)S.n, before, want);
  if (!ranked) {
    __syncthreads();
    refine<MASS>(S, row, D, b, before, want, thr_x, thr_i);
  }
  thr_x = key_logit(S.key), thr_i = key_index(S.key);
  return ranked;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs A) {
  __shared__ Shared S;
  extern __shared__ uint4 s_row[];
  const int r = blockIdx.x, tid = threadIdx.x;
  using R = Row<T>;
  constexpr int E = R::E;
  R row;
  row.l = static_cast<const T*>(A.logits) + (int64_t)r * A.ls;
  row.kept = s_row, row.V = A.V, row.odd = false, row.top = 0.f;
  row.pieces = A.pieces, row.resident = A.resident;
  const float* noise = A.noise ? A.noise + (int64_t)r * A.ns : nullptr;
  const float t0 = A.tv ? A.tv[r] : A.t, top_p = A.pv ? A.pv[r] : A.p, min_p = A.mv ? A.mv[r] : A.m;
  const int k = A.kv ? A.kv[r] : A.k;
  const bool greedy = !(t0 > 0.f);
  const bool by_k = !greedy && k > 0 && k < A.V, by_p = !greedy && top_p < 1.f;
  for (int i = tid; i < kBins; i += kThreads) S.cnt[i] = 0, S.w[i] = 0;
  if (tid == 0) S.n = 0, S.flag = 0, S.index = A.V;
  __syncthreads();

  // the largest logit; whether the row holds NaN.  Four pieces' loads in flight.
  float mine = -INFINITY;
  bool nan = false;
#pragma unroll 1
  for (int it = 0; it < row.pieces; it += 4) {
    uint4 c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = row.fetch(it + u);  // (a piece past the row is -inf)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (it + u < row.resident) row.kept[(it + u) * kThreads + tid] = c[u];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float a = Elem<T>::get(c[u], e), b = Elem<T>::get(c[u], e + 1);
        nan |= __builtin_isunordered(a, b);
        asm("v_max3_f32 %0, %1, %2, %0" : "+v"(mine) : "v"(a), "v"(b));
      }
    }
  }
  if (nan) S.flag = 1;
  float mx = block_max(S, 0, nan ? -INFINITY : mine);
  if (S.flag || mx == INFINITY) {  // uniform, rare
    if (S.flag) {
      mine = -INFINITY;
      row.each([&](const float* x, int) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine = x[e] > mine ? x[e] : mine;
      });
      mx = block_max(S, 2, mine);
    }
    row.odd = true, row.top = mx;
    if (mx == INFINITY) mine = mine == INFINITY ? 0.f : -INFINITY, mx = 0.f;
  }
  if (!(mx > -INFINITY)) {
    if (tid == 0) A.tokens[r] = -1, A.logprobs[r] = -INFINITY;
    return;
  }
  Dist D;
  D.mx = mx, D.t = greedy ? 1.f : fminf(t0, 1e30f), D.ct = fminf(KDN_LOG2E / D.t, 1e38f);

  // Few candidates: the k-th of the threads' largest logits bounds the k-th of the row from below
  float bound = INFINITY;  // log2 p of the candidates is above it
  if (by_k && k <= kFew) {
    if (mine > -INFINITY) atomicAdd(&S.cnt[first_digit(D.log2p(mine))], 1u);
    __syncthreads();
    pick_digit(S, S.cnt, 0, (u64)k);
    if (S.digit >= 0 && S.digit < kBins - 1) bound = (float)(S.digit + 1) * (-1.f / 32.f);
    for (int i = tid; i < kBins; i += kThreads) S.cnt[i] = 0;  // (read by pick_digit before its barriers)
  }
  // The whole mass, and the candidates, or where there can be none the first histogram: top-k's of the counts (and top-p's
  // of the masses), or top-p's with what is known of the whole mass before it (at least 1, the largest token's).
  const bool many = by_k && k > kFew, weigh = by_p && !by_k;
  float total = 0.f;
  if (many || weigh) {
    // log2 of p above which tokens are counted (rounded down; -inf: all that can be drawn)
    const float above = many ? -INFINITY : __log2f(0.999f * (1.f - top_p) / (float)A.V) - 0.01f;
    row.each([&](const float* x, int) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = D.log2p(x[e]), p = fexp2(y);
        total += p;
        if (y > above) {
          const int d = first_digit(y);
          if (many) atomicAdd(&S.cnt[d], 1u);
          if (by_p) atomicAdd(&S.w[d], mass_of(p));
        }
      }
    });
  } else {
    row.each([&](const float* x, int i) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = D.log2p(x[e]);
        total += fexp2(y), any |= y > bound;
      }
      if (!any) return;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = D.log2p(x[e]);
        if (y > bound) {
          const uint32_t at = atomicAdd(&S.n, 1u);
          if (at < (uint32_t)kList) S.list[at] = key_of(x[e], i + e), S.listw[at] = mass_of(fexp2(y));
        }
      }
    });
  }
  total = block_add(S, 1, total);

  float best = -1.f, top = -1.f;
  int bi = A.V;
  const int n = (int)S.n;
  if (bound < INFINITY && n <= kList) {
    rank_list(S, n);
    u64 key = 0, before = 0, w = 0;
    int rank = 0;
    if (tid < n) key = S.list[tid], w = S.listw[tid], rank = (int)S.rank[tid], before = S.run[tid];
    bool keep = tid < n && rank < k;
    if (by_p) {
      const u64 kept = block_add(S, keep ? w : 0ull);
      const double want = ceil((double)fmaxf(top_p, 0.f) * (double)kept);
      keep = keep && (before < (u64)want || rank == 0);
    }
    if (keep) {
      const float p = D.prob(key_logit(key));
      bi = key_index(key);
      best = p >= min_p ? p / noise[bi] : -1.f;
    }
    top = block_max(S, 0, best);
  } else {
    // the last token that stays, by the order
    float thr_x = -INFINITY, kept = total;
    int thr_i = -1;
    bool weighed = weigh;  // S.w holds the mass of the first digits
    u64 kept_mass = 0;
    if (by_k) {
      if (!many) {  // the candidates did not fit the list
        row.each([&](const float* x, int) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float y = D.log2p(x[e]);
            if (y > -INFINITY) {
              const int d = first_digit(y);
              atomicAdd(&S.cnt[d], 1u);
              if (by_p) atomicAdd(&S.w[d], mass_of(fexp2(y)));
            }
          }
        });
        __syncthreads();
      }
      pick_digit(S, S.cnt, 0, (u64)k);
      weighed = by_p;
      if (S.digit >= 0) {  // otherwise fewer than k can be drawn
        const int b = S.digit;
        const bool ranked = select_key<false>(S, row, D, (u64)k, thr_x, thr_i);
        if (by_p && ranked) {  // the kept mass: of the digits before, and of the list down to the threshold
          u64 m = (2 * tid < b ? S.w[2 * tid] : 0ull) + (2 * tid + 1 < b ? S.w[2 * tid + 1] : 0ull);
          if (tid < (int)S.n && S.list[tid] >= S.key) m += mass_of(fexp2(D.log2p(key_logit(S.list[tid]))));
          kept_mass = block_add(S, m);
        } else if (by_p) {  // refine has used S.w
          weighed = false;
          kept = 0.f;
          row.each([&](const float* x, int i) {
#pragma unroll
            for (int e = 0; e < E; ++e) kept += stays(x[e], i + e, thr_x, thr_i) ? fexp2(D.log2p(x[e])) : 0.f;
          });
          kept = block_add(S, 0, kept);
          for (int i = tid; i < kBins; i += kThreads) S.w[i] = 0;
          __syncthreads();
        }
      }
    }
    if (by_p) {
      // the first tokens whose mass reaches top_p of the kept mass, at least one
      const double of = kept_mass ? (double)kept_mass : (double)kept * 1099511627776.0;
      const double want_d = ceil((double)fmaxf(top_p, 0.f) * of);
      const u64 want = want_d < 1.0 ? 1ull : (u64)want_d;
      if (!weighed) {
        const float least = 0.999f * (1.f - top_p) * kept / (float)A.V;
        row.each([&](const float* x, int i) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float y = D.log2p(x[e]), p = fexp2(y);
            if (p >= least && stays(x[e], i + e, thr_x, thr_i)) atomicAdd(&S.w[first_digit(y)], mass_of(p));
          }
        });
        __syncthreads();
      }
      pick_digit(S, S.w, 0, want);
      if (S.digit >= 0)  // otherwise rounding alone keeps the sum below: all stay
        select_key<true>(S, row, D, want, thr_x, thr_i);
    }
    // The draw: each thread's best by fast arithmetic, compared between the threads by the exact quotient.  With the mass
    // m that stays, max p / e is m / Exp(1), below m / 16 once in 10^7 rows: only tokens above that (about 16 of a row)
    // are looked at closely, and all of them in a second pass if there are none.
    float from = 0.f;
    if (!(min_p > 0.f)) {
      if (by_p)
        from = fmaxf(top_p, 0.f) * (kept_mass ? (float)kept_mass / kMassOne : kept);
      else
        from = by_k ? total * ((float)k / (float)A.V) : total;
    }
    from = fmaxf(from, 1.f) * (1.f / 16);  // (the largest token's mass is 1)
    while (!greedy) {
      const float least = min_p * 0.999f;
      float score = from;
      auto offer = [&](float x, int i, float q) {
        const float p = fexp2(D.log2p(x));
        if (!(p > score * q) || !stays(x, i, thr_x, thr_i)) return;
        const float s = p * frcp(q);
        if (s > score && p >= least && (p >= min_p * 1.001f || D.prob(x) >= min_p)) score = s, bi = i;
      };
      // the noise of four pieces (those that hold a token that stays) loaded at once
      constexpr int U = 4;
#pragma unroll 1
      for (int it = 0; it < row.pieces; it += U) {
        float4 q[U][E / 4];
        bool have[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          have[u] = false;
          if (it + u >= row.pieces) continue;  // uniform
          float x[E];
          row.unpack(row.piece(it + u), x);
          float high = -INFINITY;
#pragma unroll
          for (int e = 0; e < E; e += 2) asm("v_max3_f32 %0, %1, %2, %0" : "+v"(high) : "v"(x[e]), "v"(x[e + 1]));
          have[u] = high >= thr_x && high > -INFINITY;
          if (!have[u]) continue;
          const int i = ((it + u) * kThreads + tid) * E;
          if (i + E <= A.V) {
#pragma unroll
            for (int e = 0; e < E / 4; ++e) q[u][e] = __builtin_bit_cast(float4, load16(noise + i + 4 * e));
          } else {
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
              float f[4];
#pragma unroll
              for (int h = 0; h < 4; ++h) f[h] = i + 4 * e + h < A.V ? noise[i + 4 * e + h] : 1.f;
              q[u][e] = float4{f[0], f[1], f[2], f[3]};
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!have[u]) continue;
          float x[E];
          row.unpack(row.piece(it + u), x);
          const int i = ((it + u) * kThreads + tid) * E;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float4 v = q[u][e / 4];
            offer(x[e], i + e, e % 4 == 0 ? v.x : e % 4 == 1 ? v.y : e % 4 == 2 ? v.z : v.w);
          }
        }
      }
      if (bi < A.V) best = D.prob(row.logit(bi)) / noise[bi];
      top = block_max(S, 0, best);
      if (top >= 0.f || from == 0.f) break;  // uniform
      from = 0.f;
      __syncthreads();
    }
  }
  if (!greedy) {
    if (best == top && top >= 0.f) atomicMin(&S.index, bi);
    __syncthreads();
  }
  if (S.index >= A.V) {  // uniform: greedy, or nothing has a score (noise or settings out of their ranges)
    __syncthreads();
    int at = A.V;
    row.each([&](const float* x, int i) {
#pragma unroll
      for (int e = 0; e < E; ++e) at = x[e] == mx && i + e < at ? i + e : at;
    });
    if (at < A.V) atomicMin(&S.index, at);
    __syncthreads();
  }
  if (tid == 0) {
    const int token = S.index;
    A.tokens[r] = token;
    A.logprobs[r] = D.z(row.logit(token)) - logf(total);
  }
}

template <typename T>
int launch_sample(SampleArgs A, int rows, hipStream_t stream) {
  const int per = kThreads * (16 / (int)sizeof(T));
  A.pieces = (A.V + per - 1) / per;
  A.resident = A.pieces < kResident ? A.pieces : kResident;
  const size_t lds = (size_t)A.resident * kThreads * 16;
  if (lds > 32768) {  // static and dynamic shared memory above the default limit
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&sample_kernel<T>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return (int)e;
  }
  // a launch's threads are counted in 32 bits (of more rows the remainder alone would run)
  constexpr int64_t kRows = 1 << 21;
  for (int64_t r0 = 0; r0 < rows; r0 += kRows) {
    SampleArgs P = A;
    P.logits = static_cast<const T*>(A.logits) + r0 * A.ls, P.noise = A.noise ? A.noise + r0 * A.ns : nullptr;
    P.tv = A.tv ? A.tv + r0 : nullptr, P.kv = A.kv ? A.kv + r0 : nullptr;
    P.pv = A.pv ? A.pv + r0 : nullptr, P.mv = A.mv ? A.mv + r0 : nullptr;
    P.tokens = A.tokens + r0, P.logprobs = A.logprobs + r0;
    hipLaunchKernelGGL(sample_kernel<T>, dim3((unsigned)(rows - r0 < kRows ? rows - r0 : kRows)), dim3(kThreads), lds, stream, P);
  }
  KDN_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int kdn_sample(const void* logits, int logits_dtype, int64_t logits_row_stride, const float* noise,
                          int64_t noise_row_stride, const float* temperatures, float temperature, const int* top_ks, int top_k,
                          const float* top_ps, float top_p, const float* min_ps, float min_p, int rows, int vocab,
                          int64_t* tokens, float* logprobs, hipStream_t stream) {
  if (rows < 0 || vocab < 1 || vocab > (1 << kIdxBits) || logits_dtype < 0 || logits_dtype > 2) return KDN_ERR_ARG;
  if (rows == 0) return 0;
  if (!logits || !tokens || !logprobs || (!noise && (temperatures || temperature != 0.f))) return KDN_ERR_ARG;
  if (rows > 1 && (logits_row_stride < vocab || (noise && noise_row_stride < vocab))) return KDN_ERR_ARG;
  if (!temperatures && !(temperature >= 0.f && temperature < INFINITY)) return KDN_ERR_ARG;
  if (!top_ps && !(top_p > 0.f)) return KDN_ERR_ARG;
  if (!min_ps && !(min_p >= 0.f && min_p <= 1.f)) return KDN_ERR_ARG;
  const SampleArgs A{logits, logits_row_stride, noise, noise_row_stride, temperatures, temperature, top_ks, top_k,
                     top_ps, top_p, min_ps, min_p, vocab, 0, 0, tokens, logprobs};
  if (logits_dtype == 0) return launch_sample<float>(A, rows, stream);
  if (logits_dtype == 1) return launch_sample<bf16_t>(A, rows, stream);
  return launch_sample<Half>(A, rows, stream);
}
