// Per-head norm of queries and keys with the position rotation in the same pass, and optionally the key's and value's
// way into a paged cache.
//
//   y = x * rsqrt(c * sum x^2 + eps) * w * s      (c = 1/hd: rms; c = 1: l2; no norm: y = x * s)
//   pairs (i, i + rot/2) or (2i, 2i + 1) of the first rot values:  (y1 cos - y2 sin, y1 sin + y2 cos)
//
// Bound: HBM (each head row read once, written once; 32 bits from the load to the one rounding at the store).  A group of
// lanes holds one head row, 8 values per lane through 16-byte accesses (or value by value where sizes, strides or
// pointers are no multiples of 16 bytes).  A lane keeps the same place in the row for all heads of its token, so the
// token's cosines and sines are loaded once into registers; the weights sit in shared memory.  Four head rows per group are
// in flight while four are computed.  The half layout fetches the partner value from its lane where rot / 2 is a multiple of
// 8 values, else through shared memory (padded by one word in eight: no bank conflicts), which works for every rot.
#include "common.cuh"

namespace hb200 {
namespace {

constexpr int kThreads = 128;

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
  int S, Hq, Hkv, hd, rot, page_size, group_lanes, parts, pos64;
  float norm_c, eps, q_scale, k_scale;
  int norm;
};

// Eight values of a row as they come from memory.
template <typename T, bool VEC>
struct Raw {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, int) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = __ldg(reinterpret_cast<const uint4*>(p) + j);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Cvt<T>::to_f(e[i]);
  }
  __device__ __forceinline__ void copy(T* p, int) const {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(p)[j] = v[j];
  }
};
template <typename T>
struct Raw<T, false> {
  T v[8];
  __device__ __forceinline__ void load(const T* p, int n) {
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
  __device__ __forceinline__ void copy(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
};
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float (&f)[8]) {
  Raw<T, VEC> r;
  T* e = reinterpret_cast<T*>(r.v);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = Cvt<T>::from_f(f[i]);
  r.copy(p, n);
}

// VEC: rows by 16-byte accesses.  TAB: tables by 16-byte loads, a lane's values all turned or all kept, partners in one lane.
// HALF: pairs (i, i + rot/2); else (2i, 2i + 1).  CACHE: k and v rows go to their slots, else k rows to k_out.
template <typename T, bool VEC, bool TAB, bool HALF, bool CACHE>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;                // rows in flight per group, and as many in computation
  constexpr int NC = HALF || !TAB ? 8 : 4;                 // cosines per lane
  extern __shared__ float s_rows[];
  __shared__ __align__(16) float s_w[2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int LG = p.group_lanes, groups = 32 / LG;          // lanes per head row (a power of two), rows per warp
  const int gl = lane & (LG - 1), grp = lane / LG;
  const int e0 = gl * 8;                                    // first value of this lane
  const int mine = p.hd - e0 < 8 ? (p.hd - e0 > 0 ? p.hd - e0 : 0) : 8;
  const int half = p.rot >> 1;
  float* row = s_rows + (warp * groups + grp) * (LG * 9);
  const int rows = p.Hq + p.Hkv + (CACHE ? p.Hkv : 0);
  const int step = groups * p.parts;
  for (int i = threadIdx.x; i < 256; i += kThreads) {
    s_w[0][i] = p.q_scale * (p.wq && i < p.hd ? __ldg(p.wq + i) : 1.f);
    s_w[1][i] = p.k_scale * (p.wk && i < p.hd ? __ldg(p.wk + i) : 1.f);
  }
  __syncthreads();

  const int64_t items = p.tokens * p.parts, stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + warp; item < items; item += stride) {
    const int64_t tok = p.parts == 1 ? item : item / p.parts;
    const int part = (int)(item - tok * p.parts);          // which share of the token's heads
    const int64_t b = tok < p.S ? 0 : tok / p.S, s = tok - b * p.S;
    const T* qb = static_cast<const T*>(p.q) + b * p.q_s[0] + s * p.q_s[1] + e0;
    const T* kb = static_cast<const T*>(p.k) + b * p.k_s[0] + s * p.k_s[1] + e0;
    const T* vb = CACHE ? static_cast<const T*>(p.v) + b * p.v_s[0] + s * p.v_s[1] + e0 : nullptr;
    Raw<T, VEC> raw[U], next[U];
    auto fetch = [&](Raw<T, VEC> (&x)[U], int r0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * step + grp;
        const T* src = r < p.Hq ? qb + (int64_t)r * p.q_s[2]
                                : (!CACHE || r < p.Hq + p.Hkv ? kb + (int64_t)(r - p.Hq) * p.k_s[2] : vb + (int64_t)(r - p.Hq - p.Hkv) * p.v_s[2]);
        if (r < rows && mine > 0) x[u].load(src, mine);
        else x[u].clear();
      }
    };
    fetch(raw, part * groups);

    int64_t pos = s;
    if (p.positions)
      pos = p.pos64 ? __ldg(static_cast<const long long*>(p.positions) + b * p.pos_sb + s)
                    : (int64_t)__ldg(static_cast<const int32_t*>(p.positions) + b * p.pos_sb + s);
    int64_t slot = -1;
    if constexpr (CACHE) slot = __ldg(reinterpret_cast<const long long*>(p.slots) + tok);
    const bool pad = pos < 0;                              // a row of padding: zeros out, nothing into the cache
    bool wrong = pos >= p.table_rows;                      // no angle for it: NaN, not a silent clamp
    if constexpr (CACHE) wrong |= slot >= p.capacity;
    const int64_t tr = pad || pos >= p.table_rows ? 0 : pos;

    // cosines and (signed) sines of the lane's values
    float c[NC], n[NC];
    const float* ct = p.cos_t + tr * p.table_ld;
    const float* st = p.sin_t + tr * p.table_ld;
    const bool turn = e0 < p.rot;                          // TAB: of all the lane's values
    if constexpr (TAB) {
#pragma unroll
      for (int i = 0; i < NC; ++i) c[i] = n[i] = 0.f;
      if (turn) {
        const int at = HALF ? (e0 < half ? e0 : e0 - half) : e0 >> 1;
        const float sign = HALF && e0 < half ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(ct + at + i)), d = __ldg(reinterpret_cast<const float4*>(st + at + i));
          c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
          n[i] = sign * d.x; n[i + 1] = sign * d.y; n[i + 2] = sign * d.z; n[i + 3] = sign * d.w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        c[i] = 1.f;
        n[i] = 0.f;
        if (e < p.rot) {
          const int at = HALF ? (e < half ? e : e - half) : e >> 1;
          const bool first = HALF ? e < half : (e & 1) == 0;
          c[i] = __ldg(ct + at);
          n[i] = first ? -__ldg(st + at) : __ldg(st + at);
        }
      }
    }

    T* qo = static_cast<T*>(p.q_out) + b * p.qo_s[0] + s * p.qo_s[1] + e0;
    T *ko = nullptr, *vo = nullptr;
    int64_t ko_h, vo_h = 0;
    const bool into_cache = CACHE && !pad && slot >= 0 && slot < p.capacity;
    if constexpr (CACHE) {
      const int64_t page = into_cache ? slot / p.page_size : 0, off = into_cache ? slot - page * p.page_size : 0;
      ko = static_cast<T*>(p.kc) + page * p.kc_s[0] + off * p.kc_s[2] + e0;
      vo = static_cast<T*>(p.vc) + page * p.vc_s[0] + off * p.vc_s[2] + e0;
      ko_h = p.kc_s[1];
      vo_h = p.vc_s[1];
    } else {
      ko = static_cast<T*>(p.k_out) + b * p.ko_s[0] + s * p.ko_s[1] + e0;
      ko_h = p.ko_s[2];
    }

    for (int r0 = part * groups; r0 < rows; r0 += step * U) {   // uniform over the warp
      if (r0 + step * U < rows) fetch(next, r0 + step * U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * step >= rows) break;                  // uniform over the warp
        const int r = r0 + u * step + grp;
        const bool is_q = r < p.Hq, is_v = CACHE && r >= p.Hq + p.Hkv;
        float y[8], z[8];
        raw[u].get(y);
        float inv = 1.f;
        if (p.norm) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            if (o < LG) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          inv = rsqrtf(ss * p.norm_c + p.eps);
        }
        if (wrong) inv = __int_as_float(0x7fc00000);
        const float4* w4 = reinterpret_cast<const float4*>(s_w[is_q ? 0 : 1] + e0);
        const float4 wa = w4[0], wb = w4[1];
        const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= inv * w[i];
        if constexpr (HALF && TAB) {
          const int away = half >> 3;                      // lanes between partners
          const int partner = turn ? (e0 < half ? lane + away : lane - away) : lane;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(0xffffffffu, y[i], partner);
            z[i] = turn ? fmaf(y[i], c[i], other * n[i]) : y[i];
          }
        } else if constexpr (HALF) {
          __syncwarp();                                    // the row before this one has been read
#pragma unroll
          for (int i = 0; i < 8; ++i) row[gl * 9 + i] = y[i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int e = e0 + i;
            const int other = e < half ? e + half : e - half;
            z[i] = e < p.rot ? fmaf(y[i], c[i], row[(other >> 3) * 9 + (other & 7)] * n[i]) : y[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float cc = TAB ? c[i / 2] : c[i], first = TAB ? -n[i / 2] : n[i], second = TAB ? n[i / 2] : n[i + 1];
            const bool in = TAB ? turn : e0 + i < p.rot;   // rot is even: a pair is turned or kept as a whole
            z[i] = in ? fmaf(y[i], cc, y[i + 1] * first) : y[i];
            z[i + 1] = in ? fmaf(y[i + 1], cc, y[i] * second) : y[i + 1];
          }
        }
        if (r < rows && mine > 0) {
          if (pad) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = 0.f;
          }
          if (is_q) {
            store8<T, VEC>(qo + (int64_t)r * p.qo_s[2], mine, z);
          } else if (!CACHE) {
            store8<T, VEC>(ko + (int64_t)(r - p.Hq) * ko_h, mine, z);
          } else if (into_cache) {
            if (is_v) raw[u].copy(vo + (int64_t)(r - p.Hq - p.Hkv) * vo_h, mine);
            else store8<T, VEC>(ko + (int64_t)(r - p.Hq) * ko_h, mine, z);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
    }
  }
}

template <typename T, bool VEC, bool TAB, bool HALF, bool CACHE>
int launch_as(const RopeParams& p, cudaStream_t st) {
  int dev = 0, sms = 0;
  HB_CUDA(cudaGetDevice(&dev));
  HB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  int64_t grid = ceil_div64(p.tokens * p.parts, kThreads / 32);
  if (grid > (int64_t)sms * 16) grid = (int64_t)sms * 16;
  qk_norm_rope_kernel<T, VEC, TAB, HALF, CACHE><<<(unsigned)grid, kThreads, HALF && !TAB ? kThreads * 9 * 4 : 0, st>>>(p);
  HB_LAUNCH_CHECK();
  return 0;
}

template <typename T, bool HALF, bool CACHE>
int launch_mode(const RopeParams& p, bool vec, bool tab, cudaStream_t st) {
  if (!vec) return launch_as<T, false, false, HALF, CACHE>(p, st);
  return tab ? launch_as<T, true, true, HALF, CACHE>(p, st) : launch_as<T, true, false, HALF, CACHE>(p, st);
}

template <typename T>
int launch(const RopeParams& p, bool vec, bool tab, bool half, bool cache, cudaStream_t st) {
  if (half) return cache ? launch_mode<T, true, true>(p, vec, tab, st) : launch_mode<T, true, false>(p, vec, tab, st);
  return cache ? launch_mode<T, false, true>(p, vec, tab, st) : launch_mode<T, false, false>(p, vec, tab, st);
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
  HB_REQUIRE(a->table_rows >= 0 && a->table_ld >= a->rot / 2, HB200_ERR_INVALID, "qk_norm_rope: bad table shape");
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
  p.group_lanes = 1;
  while (p.group_lanes * 8 < p.hd) p.group_lanes <<= 1;
  // a token's head rows are shared out over `parts` warps until about 16 warps per SM have work
  const int rows = a->Hq + a->Hkv * (c ? 2 : 1), groups = 32 / p.group_lanes;
  p.parts = 1;
  while (tokens * p.parts < 148 * 16 && p.parts * groups < rows) p.parts <<= 1;
  const bool tab = a->rot % (a->layout == HB200_ROPE_HALF ? 16 : 8) == 0 && a->table_ld % 4 == 0 && aligned16(a->cos) && aligned16(a->sin);
  cudaStream_t st = (cudaStream_t)stream;
  const bool half = a->layout == HB200_ROPE_HALF;
  if (a->dtype == HB200_F32) return launch<float>(p, vec, tab, half, c != nullptr, st);
  if (a->dtype == HB200_BF16) return launch<__nv_bfloat16>(p, vec, tab, half, c != nullptr, st);
  if (a->dtype == HB200_F16) return launch<__half>(p, vec, tab, half, c != nullptr, st);
  set_error("qk_norm_rope: unsupported dtype %d", a->dtype);
  return HB200_ERR_UNSUPPORTED;
}
