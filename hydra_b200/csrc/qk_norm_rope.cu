// Per-head norm of queries and keys with the position rotation in the same pass, and optionally the key's and value's
// way into a paged cache.
//
//   y = x * rsqrt(c * sum x^2 + eps) * w * s      (c = 1/hd: rms; c = 1: l2; no norm: y = x * s)
//   pairs (i, i + rot/2) or (2i, 2i + 1) of the first rot values:  (y1 cos - y2 sin, y1 sin + y2 cos)
//
// Bound: HBM (each head row read once, written once; 32 bits from the load to the one rounding at the store).  A group of
// lanes takes one token's queries, keys or values (or a part of them where there are few tokens), head row after head row,
// 8 values per lane through 16- or 8-byte accesses (or value by value where sizes, strides or pointers are no multiples of
// 16 bytes).  A lane keeps the same place in the row for all heads, so the products of the token's cosines and sines with the
// weights sit in its registers, and a head row costs two packed products and a fused one per pair of values; the norm's factor is
// the same for the whole row and comes last.  Four head rows per group are in flight while four are computed.  In the half
// layout a lane holds four values and their four partners where rot is a multiple of 8; else partners meet in shared memory.
// Measured (device time): 32768 tokens of 32 + 8 + 8 heads of 128 into a cache: 132 us, 6.1 TB/s, 0.94 of a copy; 16384 of them in
// fp32, the same bytes: 126.
#include "common.cuh"

namespace hb200 {
namespace {

// A warp per CTA: nothing is shared between warps, and a finished one makes room at once (32768 tokens of 48 heads of 128: 132 us;
// 64 threads: 141, 128: 142, 256: 161).
constexpr int kThreads = 32;

struct RopeParams {
  const void *q, *k, *v;
  void *q_out, *k_out, *kc, *vc;
  const int64_t* slots;
  const void* positions;
  const float *cos_t, *sin_t, *wq, *wk;
  int64_t q_s[3], k_s[3], v_s[3];        // batch, token, head
  int64_t qo_s[3], ko_s[3];
  int64_t kc_s[3], vc_s[3];              // page, head, row
  int64_t tokens, pos_sb, table_ld, table_rows, capacity;
  int64_t q_warps, kv_warps;             // warps' worth of query items, of key (and of value) items
  int S, Hq, Hkv, hd, rot, page_size, group_lanes, q_parts, kv_parts, pos64;
  float norm_c, eps, q_scale, k_scale;
  int norm;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2_rn(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Eight values of a row as they come from memory: one after another, or (SPLIT) four and four, `gap` apart.
template <typename T, bool VEC, bool SPLIT>
struct Raw {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ void load(const T* p, int gap, int) {
    if constexpr (sizeof(T) == 4 || !SPLIT) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(SPLIT && j ? p + gap : p) + (SPLIT ? 0 : j));
        w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
      }
    } else {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(p)), b = __ldg(reinterpret_cast<const uint2*>(p + gap));
      w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 2 * (int)sizeof(T); ++j) w[j] = 0;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Cvt<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void copy(T* p, int gap, int) const {
    if constexpr (sizeof(T) == 4 || !SPLIT) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j)
        *(reinterpret_cast<uint4*>(SPLIT && j ? p + gap : p) + (SPLIT ? 0 : j)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + gap) = make_uint2(w[2], w[3]);
    }
  }
};
template <typename T>
struct Raw<T, false, false> {
  T v[8];
  __device__ __forceinline__ void load(const T* p, int, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : Cvt<T>::from_f(0.f);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Cvt<T>::from_f(0.f);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Cvt<T>::to_f(v[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Cvt<T>::from_f(f[i]);
  }
  __device__ __forceinline__ void copy(T* p, int, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
};

// Two 32-bit values in one operation.
struct F2 {
  uint64_t v;
  __device__ F2() {}
  __device__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
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

// VEC: rows by 16-byte (8-byte) accesses.  FAST: a lane's values are all turned or all kept and it holds their partners, its
// angles come by 16-byte loads; else value by value, partners through shared memory.  HALF: pairs (i, i + rot/2); else
// (2i, 2i + 1).  CACHE: k and v rows go to their slots, else k rows to k_out.
template <typename T, bool VEC, bool FAST, bool HALF, bool CACHE>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;                // head rows in flight per group, and as many in computation
  constexpr bool SPLIT = HALF && FAST;                     // four values of the first half and their partners
  using R = Raw<T, VEC, SPLIT>;
  extern __shared__ __align__(16) float s_rows[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int LG = p.group_lanes, groups = 32 / LG;          // lanes per head row (a power of two), rows per warp
  const int gl = lane & (LG - 1), grp = lane / LG;
  const bool in_head = gl * 8 < p.hd;                      // (else a lane behind the head's end: it reads what lane 0 reads)
  const int half = p.rot >> 1;
  // first value of this lane, and how far from it its second four lie
  int e0 = in_head ? gl * 8 : 0, gap = 4;
  bool turn = e0 < p.rot;                                  // FAST: of all the lane's values
  if constexpr (SPLIT) {
    const int g = in_head ? gl : 0;
    turn = g * 4 < half;
    if (turn) { e0 = g * 4; gap = half; }                  // (else what is kept: rot is a multiple of 8)
  }
  const int mine = p.hd - e0 < 8 ? p.hd - e0 : 8;
  float* row = s_rows + (warp * groups + grp) * (LG * 9);

  // x of the lane's partners (what comes where a value has none is not used)
  auto partners = [&](const float (&x)[8], float (&y)[8]) {
    if constexpr (SPLIT) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i ^ 4];
    } else if constexpr (!HALF) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
    } else {                                               // one word of padding in eight: no bank conflicts
      __syncwarp();                                        // the row before this one has been read
#pragma unroll
      for (int i = 0; i < 8; ++i) row[gl * 9 + i] = x[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i, other = e < half ? e + half : (e < p.rot ? e - half : e);
        y[i] = row[(other >> 3) * 9 + (other & 7)];
      }
    }
  };

  // items: first all tokens' queries, then keys, then values; a warp's groups take neighbouring tokens and one kind
  // (a warp takes one item: a grid that fits the GPU once and walks over them was slower)
  const int64_t wi = (int64_t)blockIdx.x * (kThreads / 32) + warp;
  if (wi >= p.q_warps + p.kv_warps * (CACHE ? 2 : 1)) return;
  const int kind = wi < p.q_warps ? 0 : (wi < p.q_warps + p.kv_warps ? 1 : 2);
  const int step = kind == 0 ? p.q_parts : p.kv_parts;   // parts of a token's heads: a group takes every step-th row
  const int rows = kind == 0 ? p.Hq : p.Hkv;
  const int64_t item = (wi - (kind == 0 ? 0 : (kind == 1 ? p.q_warps : p.q_warps + p.kv_warps))) * groups + grp;
  int64_t tok = step == 1 ? item : item / step;
  const int first = (int)(item - tok * step);            // this group's first head row
  bool put = in_head && tok < p.tokens;                  // whether this lane stores anything
  if (tok >= p.tokens) tok = p.tokens - 1;               // (a group behind the last item reads the last token)
  const int64_t b = tok < p.S ? 0 : tok / p.S, s = tok - b * p.S;

  int64_t pos = s;
  if (p.positions)
    pos = p.pos64 ? __ldg(static_cast<const long long*>(p.positions) + b * p.pos_sb + s)
                  : (int64_t)__ldg(static_cast<const int32_t*>(p.positions) + b * p.pos_sb + s);
  int64_t slot = -1;
  if constexpr (CACHE) slot = __ldg(reinterpret_cast<const long long*>(p.slots) + tok);

  const int64_t* in_s = kind == 0 ? p.q_s : (kind == 1 ? p.k_s : p.v_s);
  const T* src = static_cast<const T*>(kind == 0 ? p.q : (kind == 1 ? p.k : p.v)) + b * in_s[0] + s * in_s[1] + first * in_s[2] + e0;
  const int64_t in_step = in_s[2] * step;
  R raw[U];
  const int full = rows / step / U * U;                  // rows that every group has, in whole batches
  if (full > 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(src + u * in_step, gap, mine);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * step < rows) raw[u].load(src + u * in_step, gap, mine);
      else raw[u].clear();
  }

  const bool pad = pos < 0;                              // a row of padding: zeros out, nothing into the cache
  bool wrong = pos >= p.table_rows;                      // no angle for it: NaN, not a silent clamp
  if constexpr (CACHE) wrong |= slot >= p.capacity;
  T* dst;
  int64_t out_step;
  if (CACHE && kind > 0) {
    const bool there = !pad && slot >= 0 && slot < p.capacity;
    put &= there;
    const int64_t page = there ? slot / p.page_size : 0, off = there ? slot - page * p.page_size : 0;
    const int64_t* out_s = kind == 1 ? p.kc_s : p.vc_s;
    dst = static_cast<T*>(kind == 1 ? p.kc : p.vc) + page * out_s[0] + first * out_s[1] + off * out_s[2] + e0;
    out_step = out_s[1] * step;
  } else {
    const int64_t* out_s = kind == 0 ? p.qo_s : p.ko_s;
    dst = static_cast<T*>(kind == 0 ? p.q_out : p.k_out) + b * out_s[0] + s * out_s[1] + first * out_s[2] + e0;
    out_step = out_s[2] * step;
  }

  // cw, nw: z_i = (x_i cw_i + x_partner nw_i) * factor of the norm
  F2 cw[4], nw[4];
  if (!CACHE || kind < 2) {
    const int64_t tr = wrong || pad ? 0 : pos;
    const float* ct = p.cos_t + tr * p.table_ld;
    const float* st = p.sin_t + tr * p.table_ld;
    const float* wt = kind == 0 ? p.wq : p.wk;
    const float scale = kind == 0 ? p.q_scale : p.k_scale;
    float c[8], n[8], w[8], wp[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { c[i] = 1.f; n[i] = 0.f; w[i] = scale; }
    if constexpr (FAST) {
      if (turn) {
        const int at = HALF ? e0 : e0 >> 1;
        const float4 x = __ldg(reinterpret_cast<const float4*>(ct + at)), y = __ldg(reinterpret_cast<const float4*>(st + at));
        const float a[4] = {x.x, x.y, x.z, x.w}, d[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int lower = HALF ? i : 2 * i, upper = HALF ? i + 4 : 2 * i + 1;
          c[lower] = c[upper] = a[i];
          n[lower] = -d[i];
          n[upper] = d[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        if (e < p.rot) {
          const int at = HALF ? (e < half ? e : e - half) : e >> 1;
          const bool lower = HALF ? e < half : (e & 1) == 0;
          c[i] = __ldg(ct + at);
          n[i] = lower ? -__ldg(st + at) : __ldg(st + at);
        }
      }
    }
    if (wt) {
      if (VEC && (reinterpret_cast<uintptr_t>(wt) & 15) == 0) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(wt + e0)), d = __ldg(reinterpret_cast<const float4*>(wt + e0 + gap));
        w[0] *= a.x; w[1] *= a.y; w[2] *= a.z; w[3] *= a.w;
        w[4] *= d.x; w[5] *= d.y; w[6] *= d.z; w[7] *= d.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < mine || SPLIT) w[i] *= __ldg(wt + e0 + (i < 4 ? i : gap + i - 4));
      }
    }
    partners(w, wp);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cw[i] = F2(c[2 * i] * w[2 * i], c[2 * i + 1] * w[2 * i + 1]);
      nw[i] = F2(n[2 * i] * wp[2 * i], n[2 * i + 1] * wp[2 * i + 1]);
    }
  }
  const float eps = wrong ? __int_as_float(0x7fc00000) : p.eps;
  const bool partial = p.rot < p.hd;                     // some values are kept: not even touched by a partner's inf or NaN
  // The first `left` of U head rows in place (the same number for all lanes).  First the sums of squares of all of them, whose
  // shuffles then run side by side.
  auto work = [&](R (&v)[U], int left) {
    float inv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) inv[u] = wrong ? eps : 1.f;
    if (p.norm) {
      float ss[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ss[u] = 0.f;
        if (u >= left) break;
        float x[8], sa, sb;
        v[u].get(x);
        F2 s2 = mul2(F2(x[0], x[1]), F2(x[0], x[1]));
#pragma unroll
        for (int i = 1; i < 4; ++i) s2 = fma2(F2(x[2 * i], x[2 * i + 1]), F2(x[2 * i], x[2 * i + 1]), s2);
        s2.get(sa, sb);
        ss[u] = in_head ? sa + sb : 0.f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < LG) {
#pragma unroll
          for (int u = 0; u < U; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) inv[u] = rsqrtf(fmaf(ss[u], p.norm_c, eps));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= left) break;
      float x[8], y[8], z[8];
      v[u].get(x);
      partners(x, y);
      const F2 inv2(inv[u], inv[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 a = mul2(F2(x[2 * i], x[2 * i + 1]), cw[i]);
        mul2(fma2(F2(y[2 * i], y[2 * i + 1]), nw[i], a), inv2).get(z[2 * i], z[2 * i + 1]);
        if (partial) {
          float k0, k1;
          mul2(a, inv2).get(k0, k1);
          if (FAST ? !turn : e0 + 2 * i >= p.rot) z[2 * i] = k0;
          if (FAST ? !turn : e0 + 2 * i + 1 >= p.rot) z[2 * i + 1] = k1;
        }
      }
      v[u].set(z);
      if (pad) v[u].clear();
    }
  };
  // whole batches first, without a look at the bounds; the next batch's loads are under way while one is computed
  int i = 0;
  for (; i < full; i += U) {
    R next[U];
    src += U * in_step;
    if (i + U < full) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u].load(src + u * in_step, gap, mine);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + (i + U + u) * step < rows) next[u].load(src + u * in_step, gap, mine);
        else next[u].clear();
    }
    if (!CACHE || kind < 2) work(raw, U);                // (values go as they are)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (put) raw[u].copy(dst + u * out_step, gap, mine);
      raw[u] = next[u];
    }
    dst += U * out_step;
  }
  if (i * step >= rows) return;                          // uniform over the warp
  if (!CACHE || kind < 2) work(raw, (rows - i * step + step - 1) / step);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (put && first + (i + u) * step < rows) raw[u].copy(dst + u * out_step, gap, mine);
  }
}

template <typename T, bool VEC, bool FAST, bool HALF, bool CACHE>
int launch_as(const RopeParams& p, cudaStream_t st) {
  const int64_t grid = ceil_div64(p.q_warps + p.kv_warps * (CACHE ? 2 : 1), kThreads / 32);
  HB_REQUIRE(grid <= 0x7fffffff, HB200_ERR_UNSUPPORTED, "qk_norm_rope: too many tokens");
  qk_norm_rope_kernel<T, VEC, FAST, HALF, CACHE><<<(unsigned)grid, kThreads, HALF && !FAST ? kThreads * 9 * 4 : 0, st>>>(p);
  HB_LAUNCH_CHECK();
  return 0;
}

template <typename T, bool HALF, bool CACHE>
int launch_mode(const RopeParams& p, bool vec, bool fast, cudaStream_t st) {
  if (!vec) return launch_as<T, false, false, HALF, CACHE>(p, st);
  return fast ? launch_as<T, true, true, HALF, CACHE>(p, st) : launch_as<T, true, false, HALF, CACHE>(p, st);
}

template <typename T>
int launch(const RopeParams& p, bool vec, bool fast, bool half, bool cache, cudaStream_t st) {
  if (half) return cache ? launch_mode<T, true, true>(p, vec, fast, st) : launch_mode<T, true, false>(p, vec, fast, st);
  return cache ? launch_mode<T, false, true>(p, vec, fast, st) : launch_mode<T, false, false>(p, vec, fast, st);
}

}  // namespace
}  // namespace hb200

using namespace hb200;

extern "C" int hb200_qk_norm_rope(const hb200_qk_norm_rope_args* a, const hb200_paged_cache* c, void* stream) {
  HB_REQUIRE(a, HB200_ERR_INVALID, "qk_norm_rope: null pointer");
  HB_REQUIRE(a->B >= 0 && a->S >= 0 && a->Hq >= 0 && a->Hkv >= 0 && a->hd >= 1, HB200_ERR_INVALID,
             "qk_norm_rope: bad shape B=%d S=%d Hq=%d Hkv=%d hd=%d", a->B, a->S, a->Hq, a->Hkv, a->hd);
  HB_REQUIRE(a->hd <= 256, HB200_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d (up to 256 is built)", a->hd);
  HB_REQUIRE(a->rot >= 0 && a->rot <= a->hd && a->rot % 2 == 0, HB200_ERR_INVALID,
             "qk_norm_rope: %d rotated values of a head of %d (an even number within the head)", a->rot, a->hd);
  HB_REQUIRE(a->layout == HB200_ROPE_INTERLEAVED || a->layout == HB200_ROPE_HALF, HB200_ERR_INVALID, "qk_norm_rope: unknown layout %d", a->layout);
  HB_REQUIRE(a->norm >= HB200_NORM_NONE && a->norm <= HB200_NORM_L2, HB200_ERR_INVALID, "qk_norm_rope: unknown norm %d", a->norm);
  HB_REQUIRE(a->table_rows >= (a->rot > 0 ? 1 : 0) && a->table_ld >= a->rot / 2, HB200_ERR_INVALID, "qk_norm_rope: bad table shape");
  HB_REQUIRE(a->positions || a->S <= a->table_rows, HB200_ERR_INVALID, "qk_norm_rope: tables of %lld rows for %d positions",
             (long long)a->table_rows, a->S);
  const int64_t tokens = (int64_t)a->B * a->S;
  if (tokens == 0 || a->Hq + a->Hkv == 0) return 0;
  HB_REQUIRE((a->Hq == 0 || (a->q && a->q_out)) && (a->Hkv == 0 || a->k) && (a->rot == 0 || (a->cos && a->sin)), HB200_ERR_INVALID,
             "qk_norm_rope: null pointer");
  const size_t es = a->dtype == HB200_F32 ? 4 : 2;
  RopeParams p = {};
  p.q = a->q; p.k = a->k; p.q_out = a->q_out; p.k_out = a->k_out;
  p.positions = a->positions; p.pos64 = a->positions_64; p.pos_sb = a->positions_stride;
  p.cos_t = a->cos; p.sin_t = a->sin; p.wq = a->q_weight; p.wk = a->k_weight;
  p.tokens = tokens; p.table_ld = a->table_ld; p.table_rows = a->table_rows;
  p.S = a->S; p.Hq = a->Hq; p.Hkv = a->Hkv; p.hd = a->hd; p.rot = a->rot;
  p.norm = a->norm; p.norm_c = a->norm == HB200_NORM_RMS ? 1.f / (float)a->hd : 1.f;
  p.eps = a->eps; p.q_scale = a->q_scale; p.k_scale = a->k_scale;
  bool vec = a->hd % 8 == 0;
  auto fits = [&](const void* ptr, const int64_t (&s)[3]) {
    vec = vec && aligned16(ptr);
    for (int64_t x : s) vec = vec && (x * (int64_t)es) % 16 == 0;
  };
  for (int i = 0; i < 3; ++i) {
    p.q_s[i] = a->q_stride[i]; p.k_s[i] = a->k_stride[i]; p.v_s[i] = a->v_stride[i];
    p.qo_s[i] = a->q_out_stride[i]; p.ko_s[i] = a->k_out_stride[i];
  }
  if (a->Hq) { fits(p.q, p.q_s); fits(p.q_out, p.qo_s); }
  if (a->Hkv) fits(p.k, p.k_s);
  if (c) {
    HB_REQUIRE(a->slots && a->v && c->k && c->v, HB200_ERR_INVALID, "qk_norm_rope: null pointer (cache, slots or v)");
    HB_REQUIRE(c->n_kv_heads == a->Hkv && c->head_dim == a->hd && c->dtype == a->dtype && c->num_pages >= 0 && c->page_size >= 1,
               HB200_ERR_INVALID, "qk_norm_rope: the cache's heads or dtype are not those of k");
    // Rows that share bytes, with one another or with what is read, would hold what came last.  (Keys and values may lie between
    // one another, by the same strides.)
    const int64_t size = (int64_t)es, row = a->hd * size;
    const Axis kp = {c->num_pages, c->k_stride_page * size}, kh = {c->n_kv_heads, c->k_stride_head * size}, kr = {c->page_size, c->k_stride_row * size};
    const Axis vp = {c->num_pages, c->v_stride_page * size}, vh = {c->n_kv_heads, c->v_stride_head * size}, vr = {c->page_size, c->v_stride_row * size};
    const Reach stored[] = {reach_of(c->k, row, {kp, kh, kr}), reach_of(c->v, row, {vp, vh, vr})};
    HB_REQUIRE(rows_apart(row, {kp, kh, kr}) && rows_apart(row, {vp, vh, vr}), HB200_ERR_INVALID,
               "qk_norm_rope: the cache's rows lie on top of one another");
    auto same = [](const Axis& x, const Axis& y) { return x.n < 2 || x.step == y.step; };
    const int64_t from_k_to_v = (int64_t)reinterpret_cast<uintptr_t>(c->v) - (int64_t)reinterpret_cast<uintptr_t>(c->k);
    HB_REQUIRE(!overlap(stored[0], stored[1]) ||
                   (same(kp, vp) && same(kh, vh) && same(kr, vr) && rows_apart(row, {kp, kh, kr, {2, from_k_to_v}})),
               HB200_ERR_INVALID, "qk_norm_rope: the caches of keys and values lie on top of one another");
    auto heads = [&](const void* ptr, const int64_t (&s)[3], int n) {
      return reach_of(ptr, row, {{a->B, s[0] * size}, {a->S, s[1] * size}, {n, s[2] * size}});
    };
    const int64_t angles = a->rot / 2 * 4;
    const Reach others[] = {heads(a->q, a->q_stride, a->Hq), heads(a->k, a->k_stride, a->Hkv), heads(a->v, a->v_stride, a->Hkv),
                            heads(a->q_out, a->q_out_stride, a->Hq), reach_of(a->slots, tokens * 8),
                            reach_of(a->positions, a->positions ? (int64_t)a->S * (a->positions_64 ? 8 : 4) : 0,
                                     {{a->B, a->positions_stride * (a->positions_64 ? 8 : 4)}}),
                            reach_of(a->cos, angles, {{a->table_rows, a->table_ld * 4}}), reach_of(a->sin, angles, {{a->table_rows, a->table_ld * 4}}),
                            reach_of(a->q_weight, a->q_weight ? a->hd * 4 : 0), reach_of(a->k_weight, a->k_weight ? a->hd * 4 : 0)};
    for (const Reach& w : stored)
      for (const Reach& r : others)
        HB_REQUIRE(!overlap(w, r), HB200_ERR_INVALID, "qk_norm_rope: the caches overlap the queries, keys, values or tables that are read");
    p.v = a->v; p.kc = c->k; p.vc = c->v; p.slots = a->slots;
    p.page_size = c->page_size;
    p.capacity = (int64_t)c->num_pages * c->page_size;
    p.kc_s[0] = c->k_stride_page; p.kc_s[1] = c->k_stride_head; p.kc_s[2] = c->k_stride_row;
    p.vc_s[0] = c->v_stride_page; p.vc_s[1] = c->v_stride_head; p.vc_s[2] = c->v_stride_row;
    fits(p.v, p.v_s);
    fits(p.kc, p.kc_s);
    fits(p.vc, p.vc_s);
  } else if (a->Hkv) {
    HB_REQUIRE(a->k_out, HB200_ERR_INVALID, "qk_norm_rope: null pointer");
    fits(p.k_out, p.ko_s);
  }
  HB_REQUIRE(a->dtype == HB200_F32 || a->dtype == HB200_BF16 || a->dtype == HB200_F16, HB200_ERR_UNSUPPORTED, "qk_norm_rope: unsupported dtype %d", a->dtype);
  int sms = 0;
  HB_PROPAGATE(device_sms(&sms));
  p.group_lanes = 1;
  while (p.group_lanes * 8 < p.hd) p.group_lanes <<= 1;
  // a token's head rows are shared out over more groups of lanes until about 8 warps per SM have work (8192 tokens of ten heads of
  // 32: 4.1 us; until 32 have: 6.2, each setting up its angles)
  const int groups = 32 / p.group_lanes, kinds = c ? 2 : 1;
  p.q_parts = p.kv_parts = 1;
  auto count = [&]() {
    p.q_warps = a->Hq ? ceil_div64(tokens * p.q_parts, groups) : 0;
    p.kv_warps = a->Hkv ? ceil_div64(tokens * p.kv_parts, groups) : 0;
    return p.q_warps + kinds * p.kv_warps;
  };
  while (count() < sms * 8 && (p.q_parts < a->Hq || p.kv_parts < a->Hkv)) {
    const bool q_more = p.q_parts < a->Hq && (p.kv_parts >= a->Hkv || (int64_t)p.kv_parts * a->Hq >= (int64_t)p.q_parts * a->Hkv);
    (q_more ? p.q_parts : p.kv_parts) *= 2;
  }
  const bool fast = a->rot % 8 == 0 && a->table_ld % 4 == 0 && aligned16(a->cos) && aligned16(a->sin);
  cudaStream_t st = (cudaStream_t)stream;
  const bool half = a->layout == HB200_ROPE_HALF;
  if (a->dtype == HB200_F32) return launch<float>(p, vec, fast, half, c != nullptr, st);
  if (a->dtype == HB200_BF16) return launch<__nv_bfloat16>(p, vec, fast, half, c != nullptr, st);
  return launch<__half>(p, vec, fast, half, c != nullptr, st);
}
