// Log probabilities of given tokens, entropy and the top alternatives of logit rows, from one pass over the logits.
//
//   z = x / T, m = max z, Z = sum e^{z-m};  log p(t) = z_t - m - ln Z;  H = ln Z - sum (z-m) e^{z-m} / Z
//
// Bound: HBM for many rows (each logit read once), latency for few.  Every thread keeps a running maximum with the two
// sums relative to it in 32 bits (new maxima are rare after the first pieces, so the rescaling hardly ever runs).
//
// Top alternatives without a second pass over the row: the maxima of the threads, taken over 64 groups of threads, give a
// bound that at least `top` logits reach (the top-th largest group maximum).  Each thread has noted its maximum, or where many
// alternatives are asked for those of eight stretches of its columns; only stretches that reach the bound are read again (out of L2, all of them at once), and the few
// logits found are ranked by (value, index).  Of equal logits the lowest index comes first; ties at the bound beyond the
// candidate list's size are collected in index order.  Rows that hold NaN, or more than kCand logits above the bound, take
// `top` exact selection rounds instead.
//
// Measured (device time): 8192 rows of 50257 bf16 logits and one alternative: 134 us, 6.1 TB/s, 0.94 of a copy (153 us once the
// power cap holds the clock at 1.65 GHz: then the issue slots bound it), in f16 137, 4096 rows in fp32 135; one row: 7.9 us, 64 masked rows with 20: 8.4 us,
// launch, one trip through the row and three through barriers.
//
// Few long rows are split over a cluster of CTAs, whose partial results the first CTA merges through distributed shared memory.
#include <cooperative_groups.h>

#include "common.cuh"

namespace hb200 {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCand = 512;       // candidate list of a CTA
constexpr int kMaxTop = 32;
constexpr int kGroups = 64;
constexpr int kUnroll = 4;
constexpr int kList = 512;       // those that reach the bound

struct LogprobParams {
  const void* x;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_lp;
  int64_t* top_id;
  int64_t ld, ignore;
  int cols, top, slice;   // slice: columns per CTA of a cluster
  float inv_t;
};

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Order of logits as whole numbers: larger value, larger key; -0 as +0; NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t entry(float v, int i) { return ((uint64_t)order_key(v) << 32) | (uint32_t)~i; }
__device__ __forceinline__ int entry_index(uint64_t e) { return (int)~(uint32_t)e; }

// Statistics of logits: maximum m, and sum 2^t and sum t 2^t with t = x c - ref(m) in powers of two, c = log2(e) / T.  ref is m c as
// rounded to 32 bits: one fused multiply-add per logit, and exact, since all logits are off by the same off(m) = m c - ref(m),
// which the results put right.  It is kept within kReach, where off is below one (a thread may have seen nothing but -inf);
// a row whose maximum lies beyond (logits of millions, or a temperature near nothing) is summed up again from (x - m) c.
struct Stat {
  float m, s, u;
};
constexpr float kReach = 4e6f;
__device__ __forceinline__ float ref_of(float m, float c) { return fminf(fmaxf(m * c, -kReach), kReach); }
__device__ __forceinline__ bool beyond(float m, float c) { return fabsf(m * c) > kReach; }
__device__ __forceinline__ float off_of(float m, float c) { return beyond(m, c) ? 0.f : fmaf(m, c, -(m * c)); }
__device__ __forceinline__ void rebase(Stat& a, float d) {   // to a reference that is -d larger
  d = fmaxf(d, -200.f);
  const float f = ex2f(d);
  a.u = f * fmaf(d, a.s, a.u);
  a.s *= f;
}

// Two 32-bit values in one operation.
struct F2 {
  uint64_t v;
  __device__ F2() {}
  __device__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A 16-byte piece's maximum (NaN left out), and its values.  kRaised: those far below the reach come raised to `low`, two at
// a time in their own type (a bf16 reaches that far at every temperature), so that 2^t = 0 meets a finite t and no infinity.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr bool kRaised = false;
  static __device__ __forceinline__ uint32_t low(float) { return 0; }
  static __device__ __forceinline__ float max(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ void values(const uint4& r, uint32_t, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr bool kRaised = true;
  static __device__ __forceinline__ uint32_t low(float v) { return pack_bf16x2(v, v); }
  static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __nv_bfloat162 t = __hmax2(__hmax2(as2(r.x), as2(r.y)), __hmax2(as2(r.z), as2(r.w)));
    return fmaxf(__low2float(t), __high2float(t));
  }
  static __device__ __forceinline__ void values(const uint4& r, uint32_t low, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __hmax2_nan(as2(w[i]), as2(low));
      const uint32_t b = *reinterpret_cast<const uint32_t*>(&h);
      f[2 * i] = __uint_as_float(b << 16);
      f[2 * i + 1] = __uint_as_float(b & 0xffff0000u);
    }
  }
};
template <> struct Piece<__half> {
  static constexpr bool kRaised = false;
  static __device__ __forceinline__ uint32_t low(float) { return 0; }
  static __device__ __forceinline__ __half2 as2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __half2 t = __hmax2(__hmax2(as2(r.x), as2(r.y)), __hmax2(as2(r.z), as2(r.w)));
    return fmaxf(__low2float(t), __high2float(t));
  }
  static __device__ __forceinline__ void values(const uint4& r, uint32_t, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 t = __half22float2(as2(w[i])); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
  }
};

// What a thread keeps while it reads: its maximum and the sums of its even and of its odd columns.  -inf (and anything far
// below) counts as 2^t = 0 times a finite distance; NaN stays NaN, +inf gives infinite sums.
template <typename T>
struct Running {
  float m, ref;
  uint32_t low;
  F2 c2, s, u;
  __device__ explicit Running(float c) : m(-INFINITY), ref(-kReach), low(Piece<T>::low(-2.5f * kReach / c)), c2(c, c), s(0.f, 0.f), u(0.f, 0.f) {}
  __device__ __forceinline__ void raise(float to, float c) {   // the maximum (a NaN is none)
    if (to > m) {
      m = to;
      const float next = ref_of(to, c), d = fmaxf(ref - next, -200.f), f = ex2f(d);
      const F2 f2(f, f);
      u = mul2(fma2(F2(d, d), s, u), f2);
      s = mul2(s, f2);
      ref = next;
    }
  }
  __device__ __forceinline__ void add(const uint4& raw) {
    constexpr int V = 16 / sizeof(T);
    const F2 n2(-ref, -ref);
    float f[V];
    Piece<T>::values(raw, low, f);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      F2 t = fma2(F2(f[i], f[i + 1]), c2, n2);
      float t0, t1;
      t.get(t0, t1);
      if (!Piece<T>::kRaised) {
        t0 = max_nan(t0, -200.f);
        t1 = max_nan(t1, -200.f);
        t = F2(t0, t1);
      }
      const F2 e(ex2f(t0), ex2f(t1));
      s = add2(s, e);
      u = fma2(t, e, u);
    }
  }
  __device__ __forceinline__ void add1(float f, float c) {
    const float t = max_nan(fmaf(f, c, -ref), -200.f), e = ex2f(t);
    s = add2(s, F2(e, 0.f));
    u = fma2(F2(t, 0.f), F2(e, 0.f), u);
  }
  __device__ __forceinline__ Stat stat() const {
    Stat r;
    float x, y;
    s.get(x, y);
    r.s = x + y;
    u.get(x, y);
    r.u = x + y;
    r.m = m;
    return r;
  }
};

// What a CTA of a cluster leaves for the first one.
struct Partial {
  Stat stat;
  int n;                       // entries
  uint64_t best[kMaxTop];      // in order
};

// S: stretches of a thread's columns whose maxima are kept; 0: no alternatives are asked for.
template <typename T, int NT, int S>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const LogprobParams p) {
  constexpr bool TOP = S > 0;
  constexpr int V = 16 / sizeof(T), NW = NT / 32, LPG = NT / kGroups;   // lanes per group of threads
  __shared__ Partial s_part;
  __shared__ float s_max[NW], s_sum[NW][2];
  __shared__ float s_group[kGroups];
  __shared__ uint64_t s_cand[kCand];
  __shared__ uint64_t s_best[NW];
  __shared__ float s_bound;
  __shared__ int s_count, s_listed, s_scan[NW];
  __shared__ float s_stretch[S > 1 ? S * NT : 1];
  __shared__ uint16_t s_list[S > 1 ? kList : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = blockIdx.x / C;
  const T* row = static_cast<const T*>(p.x) + r * p.ld;
  const int c0 = min(p.cols, rank * p.slice), c1 = min(p.cols, c0 + p.slice), n = c1 - c0;
  const T* x = row + c0;
  const float c = p.inv_t * kLog2e;
  const int64_t tgt = rank == 0 ? p.tokens[r] : 0;

  // values before the first 16-byte boundary, 16-byte pieces, values behind the last
  const int to_boundary = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  const int head = min(n, to_boundary), pieces = (n - head) / V, edge = head + (n - head - pieces * V);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  auto edge_at = [&](int i) { return i < head ? i : pieces * V + i; };   // i-th value outside the pieces -> its column
  // a thread's j-th piece is tid + j NT; a stretch is kUnroll `length` of them
  const int length = S > 1 ? (pieces + NT * kUnroll * S - 1) / (NT * kUnroll * (S > 0 ? S : 1)) : 0;
  Running<T> own(c);
  float far = -INFINITY;       // the maximum of the stretch so far
  int stretch = 0, batch = 0;
  int v0 = tid;
  for (; v0 + (kUnroll - 1) * NT < pieces; v0 += kUnroll * NT) {   // four pieces, one look at their maximum
    uint4 raw[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) raw[k] = __ldg(xv + v0 + k * NT);
    float mx = Piece<T>::max(raw[0]);
#pragma unroll
    for (int k = 1; k < kUnroll; ++k) mx = fmaxf(mx, Piece<T>::max(raw[k]));
    own.raise(mx, c);
    if constexpr (S > 1) {
      far = fmaxf(far, mx);
      if (++batch == length) {
        s_stretch[stretch++ * NT + tid] = far;
        far = -INFINITY;
        batch = 0;
      }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) own.add(raw[k]);
  }
  {
    uint4 raw[kUnroll - 1];
#pragma unroll
    for (int k = 0; k < kUnroll - 1; ++k)
      if (v0 + k * NT < pieces) raw[k] = __ldg(xv + v0 + k * NT);
#pragma unroll
    for (int k = 0; k < kUnroll - 1; ++k)
      if (v0 + k * NT < pieces) {
        const float mx = Piece<T>::max(raw[k]);
        if (S > 1) far = fmaxf(far, mx);
        own.raise(mx, c);
        own.add(raw[k]);
      }
  }
  if constexpr (S > 1) {
    for (; stretch < S; ++stretch, far = -INFINITY) s_stretch[stretch * NT + tid] = far;   // (its last, and what it has not)
  }
  if (tid < edge) {   // fewer than 2 V <= NT of them
    const float f = Cvt<T>::to_f(x[edge_at(tid)]);
    own.raise(f, c);
    own.add1(f, c);
  }
  const bool scored = rank == 0 && tid == 0 && tgt >= 0 && tgt < p.cols;
  const float x_tgt = scored ? Cvt<T>::to_f(row[tgt]) : 0.f;
  Stat a = own.stat();

  // the slice's maximum (on the way those of the 64 groups of threads), then its sums relative to it
  float m = a.m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (TOP && o == LPG && (lane & (LPG - 1)) == 0) s_group[tid / LPG] = m;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  if (lane == 0) s_max[warp] = m;
  if (tid == 0) s_count = s_listed = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) m = fmaxf(m, s_max[w]);
  if (beyond(m, c) && fabsf(m) < INFINITY) {     // the same for the whole CTA
    a.s = a.u = 0.f;
    for (int i = tid; i < n; i += NT) {
      const float t = max_nan((Cvt<T>::to_f(x[i]) - m) * c, -200.f), e = ex2f(t);
      a.s += e;
      a.u = fmaf(t, e, a.u);
    }
  } else {
    rebase(a, ref_of(a.m, c) - ref_of(m, c));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  if (lane == 0) { s_sum[warp][0] = a.s; s_sum[warp][1] = a.u; }
  const int want = TOP ? min(p.top, n) : 0;
  if (TOP && want > 0 && tid < kGroups) {
    // the bound: the want-th largest group maximum (at least `want` logits reach it)
    const float mine = s_group[tid];
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) {
      const float o = s_group[i];
      above += (o > mine || (o == mine && i < tid)) ? 1 : 0;
    }
    if (above == want - 1) s_bound = mine;
  }
  const bool sane = __syncthreads_or(!(a.s == a.s)) == 0;   // else NaN or +inf somewhere: the maxima say nothing
  a = {m, 0.f, 0.f};
  if (warp == 0) {
    float s = lane < NW ? s_sum[lane][0] : 0.f, u = lane < NW ? s_sum[lane][1] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    a.s = s;
    a.u = u;
  }

  if (TOP && want > 0) {
    const float bound = s_bound;
    // every logit above the bound (`equal`: or at it) into the list; the number of them, also where it overflows
    auto collect = [&](bool equal) {
      auto offer = [&](float v, int col) {
        if (v > bound || (equal && v == bound)) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kCand) s_cand[at] = entry(v, c0 + col);
        }
      };
      auto look_at = [&](int v) {
        const uint4 raw = __ldg(xv + v);
        if (Piece<T>::max(raw) >= bound) {
          const T* u = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int i = 0; i < V; ++i) offer(Cvt<T>::to_f(u[i]), head + v * V + i);
        }
      };
      if constexpr (S == 1) {              // a thread's pieces, by its whole warp
        unsigned reach = __ballot_sync(0xffffffffu, own.m > bound || (equal && own.m == bound));
        for (; reach; reach &= reach - 1)
          for (int v = warp * 32 + __ffs(reach) - 1 + lane * NT; v < pieces; v += 32 * NT) look_at(v);
      } else {                             // the stretches' pieces, by all threads
        for (int e = 0; e < S; ++e) {
          const float mx = s_stretch[e * NT + tid];
          if (mx > bound || (equal && mx == bound)) {
            const int at = atomicAdd(&s_listed, 1);
            if (at < kList) s_list[at] = (uint16_t)(e * NT + tid);
          }
        }
        __syncthreads();
        const int listed = s_listed, per = length * kUnroll;
        if (listed > kList) return kCand + 1;
        for (int i = tid; i < listed * per; i += NT) {
          const int k = i / per, e = s_list[k] / NT, v = s_list[k] % NT + (e * per + i - k * per) * NT;
          if (v < pieces) look_at(v);
        }
      }
      if (tid < edge) {
        const int col = edge_at(tid);
        offer(Cvt<T>::to_f(x[col]), col);
      }
      __syncthreads();
      return s_count;
    };
    int found = kCand + 1;
    if (sane && bound > -INFINITY) found = collect(true);
    if (sane && found > kCand) {           // many ties at the bound: those above it, then the first that equal it
      __syncthreads();
      if (tid == 0) s_count = s_listed = 0;
      __syncthreads();
      found = collect(false);
      if (found > kCand - kMaxTop) found = kCand + 1;
      for (int i0 = 0; found < want && i0 < n; i0 += NT) {   // uniform over the CTA
        const int i = i0 + tid;
        const bool eq = i < n && Cvt<T>::to_f(x[i]) == bound;
        const unsigned vote = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) s_scan[warp] = __popc(vote);
        __syncthreads();
        int at = found + __popc(vote & ((1u << lane) - 1));
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          at += w < warp ? s_scan[w] : 0;
          found += s_scan[w];
        }
        if (eq && at < want) s_cand[at] = entry(bound, c0 + i);
        found = min(found, want);
        __syncthreads();
      }
    }
    if (sane && found <= kCand) {
      for (int i = tid; i < found; i += NT) {   // rank by counting
        const uint64_t mine = s_cand[i];
        int rk = 0;
        for (int j = 0; j < found; ++j) rk += s_cand[j] > mine ? 1 : 0;
        if (rk < want) s_part.best[rk] = mine;
      }
    } else {
      // exact selection rounds: the largest entry, then the largest below the last one (NaN in column 0 is the largest number there is)
      uint64_t last = 0;
      for (int k = 0; k < want; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < n; i += NT) {
          const uint64_t e = entry(Cvt<T>::to_f(x[i]), c0 + i);
          if ((k == 0 || e < last) && e > best) best = e;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t e = __shfl_xor_sync(0xffffffffu, best, o);
          best = e > best ? e : best;
        }
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        best = s_best[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) best = s_best[w] > best ? s_best[w] : best;
        if (tid == 0) s_part.best[k] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  if (tid == 0) { s_part.stat = a; s_part.n = want; }
  __syncthreads();

  const uint64_t* mine_best = s_part.best;
  int have = want;
  if (C > 1) {
    cluster.sync();
    if (rank == 0) {
      // The slices' statistics, a slice per lane of every warp, and their entries ranked together: each thread fetches one, all on
      // their way at once (C <= 8 slices, kMaxTop places each, empty ones 0).
      Stat b = {-INFINITY, 0.f, 0.f};
      if (lane < C) b = cluster.map_shared_rank(&s_part, lane)->stat;
      uint64_t e = 0;
      if (TOP && tid < C * kMaxTop) {
        const Partial* o = cluster.map_shared_rank(&s_part, tid / kMaxTop);
        const int have_there = o->n;
        e = o->best[tid % kMaxTop];
        if (tid % kMaxTop >= have_there) e = 0;
      }
      float top_m = b.m;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
      top_m = __shfl_sync(0xffffffffu, top_m, 0);
      rebase(b, (b.m - top_m) * c + (off_of(top_m, c) - off_of(b.m, c)));   // (-inf less -inf: a NaN that counts as -200)
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        b.s += __shfl_xor_sync(0xffffffffu, b.s, o);
        b.u += __shfl_xor_sync(0xffffffffu, b.u, o);
      }
      a = {top_m, __shfl_sync(0xffffffffu, b.s, 0), __shfl_sync(0xffffffffu, b.u, 0)};
      if (TOP) {
        if (tid < C * kMaxTop) s_cand[tid] = e;
        __syncthreads();
        have = min(p.top, p.cols);
        int rk = kMaxTop;
        if (e != 0) {
          rk = 0;
          for (int q = 0; q < C; ++q)
#pragma unroll 4
            for (int j = 0; j < p.top; ++j) rk += s_cand[q * kMaxTop + j] > e ? 1 : 0;
        }
        if (rk < have) s_part.best[rk] = e;     // (its own entries have been fetched)
        __syncthreads();
      }
    }
    cluster.sync();   // no CTA leaves while its shared memory is read
  }
  if (rank != 0) return;
  const float nan = __int_as_float(0x7fc00000);
  // no logit above -inf, or NaN / +inf among them.  (Only warp 0 holds the sums.)
  if (warp > 0) return;
  const bool none = !(a.s > 0.f) || a.m == INFINITY;
  // The sum relative to the largest logit's own term, which is 2^off as the sum holds it: where one token is nearly certain, what
  // is left is a sum of small terms next to a one, not to a power that was rounded.
  const float off = off_of(a.m, c), lz2 = log2f(a.s / ex2f(off)), lz = lz2 * kLn2;
  auto logp = [&](float v) { return fmaf(v - a.m, p.inv_t, -lz); };     // ln p of a logit
  if (lane == 0) {
    float lp = nan;
    if (tgt == p.ignore) lp = 0.f;
    else if (scored && !none) lp = logp(x_tgt);
    p.logprobs[r] = lp;
    p.entropy[r] = none ? nan : (lz2 - (a.u / a.s - off)) * kLn2;
  }
  if (TOP && lane < p.top) {   // top <= 32
    const uint64_t e = lane < have ? mine_best[lane] : 0;
    p.top_id[r * p.top + lane] = lane < have ? entry_index(e) : -1;
    p.top_lp[r * p.top + lane] = lane < have && !none ? logp(key_value((uint32_t)(e >> 32))) : nan;
  }
}

template <typename T, int NT, int S>
int launch_as(const LogprobParams& p, int64_t rows, int cluster, cudaStream_t st) {
  if (cluster > 1) return launch_chained(token_logprobs_kernel<T, NT, S>, dim3((unsigned)(rows * cluster)), dim3(NT), 0, st, false, cluster, p);
  token_logprobs_kernel<T, NT, S><<<(unsigned)rows, NT, 0, st>>>(p);
  HB_LAUNCH_CHECK();
  return 0;
}

// One stretch per thread for a few alternatives, eight for more: a stretch that reaches the bound is read again (2048 rows of
// 152064 bf16 columns, 20 alternatives: 113 us with eight, 151 with one), and noting eight costs registers (8192 rows of 50257,
// one alternative: 134 us with one, 149 with eight).
template <typename T, int NT>
int launch_nt(const LogprobParams& p, int64_t rows, int cluster, cudaStream_t st) {
  if (p.top == 0) return launch_as<T, NT, 0>(p, rows, cluster, st);
  return p.top <= 4 ? launch_as<T, NT, 1>(p, rows, cluster, st) : launch_as<T, NT, 8>(p, rows, cluster, st);
}

template <typename T>
int launch(LogprobParams p, int64_t rows, cudaStream_t st) {
  // Few long rows: up to eight CTAs per row while there is an SM for each and each still has 64 KB: shorter slices cost more in
  // the cluster's barriers and the merge than they save (one row of 152064 bf16 columns: 11.4 us in one CTA, 8.4 in four;
  // 64 rows of 50257, 100 KB each: 8.1 in one, 8.9 in two).
  int cluster = 1, sms = 0;
  HB_PROPAGATE(device_sms(&sms));
  while (cluster < 8 && rows * cluster * 2 <= sms && (int64_t)p.cols * sizeof(T) / (cluster * 2) >= 65536) cluster *= 2;
  p.slice = ceil_div(ceil_div(p.cols, cluster), 64) * 64;
  // Many rows: small CTAs, whose barriers hold up little and whose fixed work per row (joining the statistics, the bound) is
  // small; few: 512 threads get a row's bytes under way sooner; between them, and for long rows of many alternatives, 256
  // (600 rows of 50257: 18 us with 256 threads, 19 with 128; 8192 rows: 139 and 134 us).
  if (rows * cluster <= 2 * sms) return launch_nt<T, 512>(p, rows, cluster, st);
  if (rows < 6 * sms || (p.top > 4 && p.cols > 65536)) return launch_nt<T, 256>(p, rows, cluster, st);
  return launch_nt<T, 128>(p, rows, cluster, st);
}

}  // namespace
}  // namespace hb200

using namespace hb200;

extern "C" int hb200_token_logprobs(const void* logits, const int64_t* tokens, int64_t rows, int cols, int64_t ld,
                                    int64_t ignore_index, float temperature, int top, float* logprobs, float* entropy,
                                    float* top_logprobs, int64_t* top_ids, int dtype, void* stream) {
  HB_REQUIRE(rows >= 0 && cols >= 1 && (ld >= cols || rows <= 1), HB200_ERR_INVALID, "token_logprobs: bad shape rows=%lld cols=%d ld=%lld",
             (long long)rows, cols, (long long)ld);
  HB_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, HB200_ERR_INVALID,
             "token_logprobs: temperature %g (1e-6 to 1e6)", temperature);
  HB_REQUIRE(top >= 0 && top <= kMaxTop, HB200_ERR_UNSUPPORTED, "token_logprobs: %d alternatives (up to %d are built)", top, kMaxTop);
  HB_REQUIRE(top <= cols, HB200_ERR_INVALID, "token_logprobs: %d alternatives of %d columns", top, cols);
  if (rows == 0) return 0;
  HB_REQUIRE(logits && tokens && logprobs && entropy && (top == 0 || (top_logprobs && top_ids)), HB200_ERR_INVALID,
             "token_logprobs: null pointer");
  HB_REQUIRE(cols <= 1 << 30, HB200_ERR_UNSUPPORTED, "token_logprobs: %d columns (up to 2^30 are built)", cols);
  HB_REQUIRE(rows <= 0x7fffffff / 8, HB200_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  const size_t es = dtype == HB200_F32 ? 4 : 2;
  HB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0, HB200_ERR_INVALID, "token_logprobs: misaligned logits");
  LogprobParams p = {};
  p.x = logits; p.tokens = tokens; p.logprobs = logprobs; p.entropy = entropy; p.top_lp = top_logprobs; p.top_id = top_ids;
  p.ld = ld; p.ignore = ignore_index; p.cols = cols; p.top = top;
  p.inv_t = (float)(1.0 / (double)temperature);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == HB200_F32) return launch<float>(p, rows, st);
  if (dtype == HB200_BF16) return launch<__nv_bfloat16>(p, rows, st);
  if (dtype == HB200_F16) return launch<__half>(p, rows, st);
  set_error("token_logprobs: unsupported dtype %d", dtype);
  return HB200_ERR_UNSUPPORTED;
}
