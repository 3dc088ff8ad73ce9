// Attention of one new token per request over a paged key-value cache, split over the caches' lengths and joined.
//
//   s_j = scale * q . k_j  (j < len),   out = sum_j e^{s_j} v_j / sum_j e^{s_j},   lse = ln sum_j e^{s_j}
//
// Bound: HBM.  Every K and V row of the valid tokens is read once (4 * hd bytes per token and kv head) for 4 * hd * group
// operations, so for groups of up to 8 query heads the tensor cores are needed only to keep the arithmetic out of the way.  tcgen05
// would want 64 or 128 rows on the accumulator's side and a TMEM round trip for the weights; the warp-level m16n8k16 is used,
// transposed (scores^T = K Q^T, out^T = V^T P^T): the tokens and the head's values are the 16 rows and the query heads the 8
// columns, so a group of up to 8 heads costs half of what 16 padded query rows cost, in registers too.  Groups of 9 to 24 take two
// or three columns, and there it is the arithmetic that bounds: half of the issue slots, few of them waiting for memory.
//
// Work split: the tiles of all (request, kv head) pairs are laid end to end and dealt out in equal contiguous shares to
// the warps of a grid that fits the GPU once (one CTA per SM), whatever the lengths are: a batch of one long and many
// short requests keeps every SM busy to the end.  Starting and finishing a pair costs a warp as much as a few tiles, so each
// pair is that much longer when the shares are cut.  The lengths live on the device; each CTA scans them itself.  A warp streams its share through a private cp.async ring that runs on across the ends of requests, so no barrier is met between
// the scan and the share's end.  A pair that lies within one share is finished by its warp.  Of the others each warp leaves
// (max, sum, unnormalised output) in 32 bits; the CTA, whose warps' shares are neighbours, adds up those of one pair, and
// what then still spans CTAs goes through the workspace to the join kernel.  All sums run in a fixed order without
// atomics: the same inputs give the same bits.
#include <cfloat>

#include "common.cuh"
#include "mma.cuh"

namespace hb200 {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ int64_t div_up(int64_t a, int b) {   // (a 64-bit division only where it takes one)
  return a <= 0x7fffffff - b ? (int64_t)(((unsigned)a + (unsigned)b - 1) / (unsigned)b) : (a + b - 1) / b;
}
constexpr int kMaxBatch = 4096;

struct PagedParams {
  const void *q, *kc, *vc;
  void* out;
  float* lse;
  const int32_t *table, *lens;
  float* part;       // [CTAs][2] parts, then [warps] of the warps' own: each [rows][hd] outputs, [rows][2] of max and sum
  int32_t* cum;      // [B + 1] places of the requests before each one
  int64_t q_sb, q_sh, k_sh, v_sh, table_ld;     // elements
  int32_t k_sp, k_sr, v_sp, v_sr;               // bytes: page and row of a page
  int B, Hq, Hkv, hd, group, q_tiles, q_tile, tile, pair_cost, warps, rows, part_floats, page_size, width, num_pages, ctas;
  float scale_log2;  // |scale| log2(e)
  uint32_t q_sign;   // flips the signs of a pair of query values where the scale is negative
  uint32_t q_keep;   // all bits; none where the scale is zero: scores of exactly 0 (and a scale of one, for the -inf of masked tokens)
};

// Measured (device time, graph replay): one request of 131072 tokens, 32 query heads on 8 kv heads of 128: 92.8 us, 5.8 TB/s,
// 0.89 of a copy; 64 requests up to 8192 tokens, 32 heads on 4 of 64: 55.3 us, 4.9 TB/s; one request of 1500 tokens: 11.1 us, of
// which 8 are the two launches and the chain lengths -> table -> tiles -> parts -> join.  What bounds the large ones: DRAM,
// after 7 us in which the rings fill, and SMs that get up to a tenth less of it than others.  All figures in this file are
// of one state of the code and one B200; those with another choice of a constant, of that code with the one constant changed.
//
// A warp's tile: 8 KB of K and V (16 KB of heads of 256, 4 KB of small ones, whose tokens cost more arithmetic per byte and get
// twice the warps: 64 requests up to 16384 tokens, 32 heads on 4 of 16: 54.9 us with eight warps, 52.2 with sixteen).  Two tiles of a
// warp are in flight while one is computed, 128 KB of a CTA; of heads of 64 one, 96 KB, which leaves room for twelve warps (64
// requests up to 8192 tokens: 55.4 us, with eight warps and two tiles 56.2).  Heads of 128 gain nothing by that, and lose where
// there is little to do (one request of 1500: 11.6 instead of 11.1).
__host__ __device__ constexpr int tile_tokens(int HD) { return HD >= 128 ? 16 : (HD == 16 ? 64 : 32); }
__host__ __device__ constexpr int warps_of(int HD) { return HD >= 256 ? 4 : (HD == 128 ? 8 : (HD == 64 ? 12 : 16)); }
__host__ __device__ constexpr int stages_of(int HD) { return HD == 64 ? 2 : 3; }
// Most query heads that are worked on together: their outputs and queries stay in a warp's registers.  Larger groups are cut
// into tiles of one size, each of which reads the keys and values again.  (Groups of 20: 82 requests of 5115 tokens on 4 kv
// heads of 80 take 175 us in one tile and 285 in two of ten, 64 requests up to 32768 on 4 of 16 145 and 228; where the second
// read comes out of the L2, 32 requests up to 8192 on two of 128, 61 and 56.)
__host__ __device__ constexpr int most_heads(int HD) { return HD >= 256 ? 8 : 24; }
// Places that a pair takes before its first tile when the shares are cut: what its start and end cost, in tiles.  (256 requests
// of 1 to 300 tokens, 32 heads on 8 of 128: 56 us with one, 50 with two, 47 with three; all of 100 tokens: 37, 39 and 39.)
__host__ __device__ constexpr int pair_cost(int HD) { return HD <= 32 ? 2 : 3; }

// Cache length of request b as the kernel reads it: what lies outside [0, width * page_size] is marked (`poison`).
__device__ __forceinline__ int clamp_len(int len, int64_t cap, bool& poison) {
  poison = (int64_t)len > cap;
  return len < 0 ? 0 : (poison ? (int)cap : len);
}

__device__ __forceinline__ void cp_async_16_zfill(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
  mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Powers of two that every weight is raised by.  A bf16 holds 2^-126 as well as 1, but both f16 summands end in steps of 2^-24: with the
// largest weight at 2^15, next to the largest f16, they reach 2^-40 of it instead of 2^-25 (a head that rests on one token
// whose own values are zero keeps those that lie 20 nats below).  Sums and outputs are raised alike, so only the sum's
// logarithm has to know.
template <typename T> struct Raise { static constexpr float kBits = 0.f; };
template <> struct Raise<__half> { static constexpr float kBits = 15.f; };

// ln sum e^{scale s} from the largest score and the sum relative to it (0 where every score is -inf).
template <typename T>
__device__ __forceinline__ float log_sum(float m, float l, float scale_log2) {
  return fmaf(m == -INFINITY ? 0.f : m, scale_log2, log2f(l) - Raise<T>::kBits) * kLn2;
}

// Two weights in T and what the rounding left of them, in T again: each is off by at most 2^-17 of itself in bf16, and in f16 by 2^-22
// of itself or, where that is more, 2^-40 of the largest.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(a, b);
  lo = pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}
template <>
__device__ __forceinline__ void split2<__half>(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// Transposes an 8x8 matrix of 16-bit values held as in a fragment (thread 4r + c/2 holds (r, c..c+1)).
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// Swizzle of a tile's 16-byte chunks: chunk c of row r lies at place c ^ swizzle(r), so that eight rows of one chunk column
// lie in eight different bank groups (ldmatrix without conflicts).  CH: chunks per row.  The same for r and r + 8.
template <int CH>
__device__ __forceinline__ int swizzle(int r) {
  return CH >= 8 ? (r & 7) : (CH == 4 ? ((r >> 1) & 3) : ((r >> 2) & 1));
}

// A place in the row of all tiles: request b, head tile h (kv head * q_tiles + tile of its query heads), tile t of n.
struct Cursor {
  int b, h, t, n, len;
  bool poison;
};

// NQ: columns of eight query heads (a tile of up to 8: 1).  P16: the page size is a multiple of 16, so that 16 tokens side by side
// share a page: one look into the table for them (64 requests, pages of 16: 55.3 us with it, 55.6 without; one
// of 131072, pages of 64: 93.3 and 93.8).
template <typename T, int HD, int NQ, bool P16>
__global__ void __launch_bounds__(warps_of(HD) * 32, 1) paged_attention_kernel(const PagedParams p) {
  constexpr int NW = warps_of(HD), TT = tile_tokens(HD), CH = HD / 8, ST = stages_of(HD);
  constexpr int ROWB = HD * 2, KBYTES = TT * ROWB, STAGE = 2 * KBYTES;
  constexpr int MT = TT / 16;                        // 16-token tiles
  constexpr int KS = HD / 16;                        // 16-value steps of a head
  constexpr int LPR = CH >= 4 ? 4 : CH;              // copies: lanes per row (64 bytes side by side)
  constexpr int RPI = 32 / LPR, R = TT / RPI;        // rows per copy instruction, rows per lane
  constexpr int CI = CH / LPR;                       // copies per row and lane
  constexpr int PC = pair_cost(HD);
  constexpr int NO = KS < 4 ? KS : 4;                // distinct swizzled offsets of the 16-value steps
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scan_buf[33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t* s_cum = reinterpret_cast<int32_t*>(smem + NW * ST * STAGE);   // [B + 1]
  int32_t* s_len = s_cum + p.B + 1;                                      // [B]
  chain_release();   // the join kernel may take its place; it waits for this grid's end before it reads anything

  // places before each request: of its tiles, and PC before those of each request that has any
  const int64_t cap = (int64_t)p.width * p.page_size;
  {
    const int per = (p.B + NW * 32 - 1) / (NW * 32);
    const int b0 = threadIdx.x * per;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = b0 + i;
      if (b < p.B) {
        const int raw = p.lens[b];
        bool poison;
        const int len = clamp_len(raw, cap, poison);
        s_len[b] = poison ? -1 - len : len;
        mine += len > 0 ? (len + TT - 1) / TT + PC : 0;
      }
    }
    int total;
    int at = block_exclusive_scan(mine, scan_buf, total);
    for (int i = 0; i < per; ++i) {
      const int b = b0 + i;
      if (b < p.B) {
        s_cum[b] = at;
        const int v = s_len[b];
        const int len = v < 0 ? -1 - v : v;
        at += len > 0 ? (len + TT - 1) / TT + PC : 0;
      }
    }
    if (threadIdx.x == 0) s_cum[p.B] = total;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b <= p.B; b += NW * 32) p.cum[b] = s_cum[b];
  }
  const int H = p.Hkv * p.q_tiles;
  const int64_t total = (int64_t)s_cum[p.B] * H;
  const int64_t share = div_up(total, p.ctas * NW);
  const int w = blockIdx.x * NW + warp;
  const int64_t begin = min((int64_t)w * share, total), end = min(begin + share, total);
  // request b, head tile h and place `at` of place v < total, and the tiles before it
  auto locate = [&](int64_t v, int& b, int& h, int& at) {
    int lo = 0, hi = p.B;   // s_cum[lo] * H <= v < s_cum[hi] * H
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)s_cum[mid] * H <= v) lo = mid; else hi = mid;
    }
    int some = 0;           // requests before it that have tiles
    for (int a = lane; a < lo; a += 32) some += s_len[a] != 0;
    some = __reduce_add_sync(0xffffffffu, some);
    const unsigned r = (unsigned)(v - (int64_t)s_cum[lo] * H), width = s_cum[lo + 1] - s_cum[lo];
    b = lo;
    h = (int)(r / width);
    at = (int)(r - h * width);
    return v - (int64_t)PC * ((int64_t)some * H + h) - min(at, PC);
  };
  Cursor cur = {};
  int left = 0;                                      // tiles to compute
  if (begin < total) {
    int64_t after = 0;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {                    // the share's last place, then its first
      int at = 0;
      const int64_t n = locate(k ? begin : end - 1, cur.b, cur.h, at);
      if (k == 0) after = n + (at >= PC ? 1 : 0);
      left = (int)(after - n);
      cur.t = max(at - PC, 0);
    }
  }
  __shared__ int s_pair[2 * NW];                     // of the warps' first and last parts: request * H + head tile, or -1
  __shared__ int s_ends[2 * NW];                     // 1: holds the pair's first tile; 2: its last
  if (lane < 2) s_pair[2 * warp + lane] = -1;

  auto enter = [&](Cursor& c) {   // request c.b's length and tiles
    c.n = s_cum[c.b + 1] - s_cum[c.b];
    c.n -= c.n > 0 ? PC : 0;
    const int v = s_len[c.b];
    c.poison = v < 0;
    c.len = v < 0 ? -1 - v : v;
  };
  auto advance = [&](Cursor& c) {   // called only while another tile follows
    if (++c.t == c.n) {
      c.t = 0;
      if (++c.h == H) {
        c.h = 0;
        do { ++c.b; enter(c); } while (c.n == 0);
      }
    }
  };
  if (left > 0) enter(cur);

  uint8_t* ring = smem + warp * ST * STAGE;
  const uint32_t ring_u = smem_u32(ring);
  if (p.hd < HD) {   // the padding chunks are never copied to: zero them once (zero times anything the ring held before)
    for (int u = lane; u < ST * STAGE / 16; u += 32) reinterpret_cast<uint4*>(ring)[u] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  // ---- producer: four lanes (two of heads of 16) copy a row; the pages are looked up one tile before the copies are issued
  constexpr int L = P16 ? MT : R;             // looks per tile: of 16 tokens each, or of each of the lane's rows
  Cursor pc = cur;
  int to_look = left, to_issue = left;
  const int unit = P16 ? p.page_size / 16 : p.page_size;      // looks per page
  int page0, off0;                            // of the tile's first token: place in the table row, units into the page
  {
    const unsigned at = (unsigned)pc.t * (P16 ? MT : TT);
    page0 = (int)(at / (unsigned)unit);
    off0 = (int)(at - (unsigned)page0 * (unsigned)unit);
  }
  const int prow = lane / LPR, pch = lane % LPR;
  const int32_t* trow = nullptr;
  const char *kb = nullptr, *vb = nullptr;    // the head's rows in page 0, from this lane's chunk on
  auto head_of = [&]() {
    const int kvh = p.q_tiles == 1 ? pc.h : pc.h / p.q_tiles;
    trow = p.table + (int64_t)pc.b * p.table_ld;
    kb = static_cast<const char*>(p.kc) + (int64_t)kvh * p.k_sh * 2 + pch * 16 + (P16 ? (int64_t)prow * p.k_sr : 0);
    vb = static_cast<const char*>(p.vc) + (int64_t)kvh * p.v_sh * 2 + pch * 16 + (P16 ? (int64_t)prow * p.v_sr : 0);
  };
  head_of();
  const char *kt = kb, *vt = vb;              // the same of the tile that was looked up
  int page[L], off[L], rows_there = 0;        // its pages, places in them, tokens
  bool bad_seen = false;                      // a page outside the cache
  uint32_t bad_bits = 0;                      // the same per ring slot
  uint32_t dst[2];                            // of the lane's even and odd copies of a row
#pragma unroll
  for (int i = 0; i < 2; ++i) dst[i] = ring_u + prow * ROWB + (((pch + (CI > 1 ? LPR * i : 0)) ^ swizzle<CH>(prow)) & (CH >= 8 ? 7 : CH - 1)) * 16;
  auto look = [&]() {
    if (to_look > 0) {
      --to_look;
      kt = kb;
      vt = vb;
      bool bad = pc.poison;
      rows_there = pc.len - pc.t * TT;        // > 0
      if constexpr (P16) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bool in = i == 0 || i * 16 < rows_there;
          page[i] = in ? __ldg(trow + page0) : 0;
          bad |= (unsigned)page[i] >= (unsigned)p.num_pages;
          off[i] = off0;
          if (++off0 == unit) { off0 = 0; ++page0; }
        }
      } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const int r = prow + j * RPI;
          int pi = page0, o = off0 + r;
          const int k = o / unit;
          pi += k;
          o -= k * unit;
          page[j] = r < rows_there ? __ldg(trow + pi) : 0;
          bad |= (unsigned)page[j] >= (unsigned)p.num_pages;
          off[j] = o;
        }
        off0 += TT;
        const int k = off0 / unit;
        page0 += k;
        off0 -= k * unit;
      }
      bad_seen = bad;
      if (to_look > 0) {
        const int b = pc.b, h = pc.h;
        advance(pc);
        if (pc.b != b || pc.h != h) {
          page0 = off0 = 0;
          head_of();
          // the next pair's queries (128 bytes a lane) come near before they are asked for
          const int qt = p.q_tiles == 1 ? 0 : pc.h % p.q_tiles, h0 = (p.q_tiles == 1 ? pc.h : pc.h / p.q_tiles) * p.group + qt * p.q_tile;
          constexpr int LPQ = (HD * 2 + 127) / 128;         // lanes per query head
#pragma unroll
          for (int i = 0; i < (NQ * 8 * LPQ + 31) / 32; ++i) {
            const int u = i * 32 + lane, r = u / LPQ;
            if (r < min(p.q_tile, p.group - qt * p.q_tile) && u % LPQ * 64 < p.hd)
              prefetch(static_cast<const T*>(p.q) + (int64_t)pc.b * p.q_sb + (int64_t)(h0 + r) * p.q_sh + u % LPQ * 64);
          }
        }
      }
    }
  };
  const int64_t k_next = (int64_t)RPI * p.k_sr, v_next = (int64_t)RPI * p.v_sr;
  auto issue = [&](int slot) {
    if (to_issue > 0) {
      --to_issue;
      const uint32_t so = slot * STAGE;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int l = P16 ? j * RPI / 16 : j;
        const bool ok = (unsigned)page[l] < (unsigned)p.num_pages;
        const bool there = ok && prow + j * RPI < rows_there;
        const int pg = ok ? page[l] : 0;
        const char* ks = kt + (int64_t)pg * p.k_sp + (int64_t)(P16 ? off[l] * 16 : off[l]) * p.k_sr;
        const char* vs = vt + (int64_t)pg * p.v_sp + (int64_t)(P16 ? off[l] * 16 : off[l]) * p.v_sr;
        if (P16 && j * RPI % 16 != 0) { ks += k_next; vs += v_next; }
#pragma unroll
        for (int i = 0; i < CI; ++i) {
          if (p.hd == HD || (pch + LPR * i) * 8 < p.hd) {
            const uint32_t d = dst[i & 1] + so + j * RPI * ROWB + (i >> 1) * 128;
            cp_async_16_zfill(d, ks + i * LPR * 16, there);
            cp_async_16_zfill(d + KBYTES, vs + i * LPR * 16, there);
          }
        }
      }
      const bool any_bad = P16 ? bad_seen : __any_sync(0xffffffffu, bad_seen);   // P16: the same in every lane
      bad_bits = any_bad ? bad_bits | (1u << slot) : bad_bits & ~(1u << slot);
    }
    cp_async_commit();
  };
  look();
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) { issue(i); look(); }

  // ---- consumer.  Fragments (g = lane / 4, t4 = lane % 4): scores^T and out^T hold rows g, g + 8 (tokens, values of the
  // head) and columns 2 t4, 2 t4 + 1 (query heads).
  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, mr = lane & 7;
  uint32_t kofs[NO], vofs[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) {
    constexpr int mask = CH >= 8 ? 7 : CH - 1;
    kofs[i] = ((mi & 1) * 8 + mr) * ROWB + (((2 * i + (mi >> 1)) ^ swizzle<CH>(mr)) & mask) * 16;
    vofs[i] = KBYTES + ((mi >> 1) * 8 + mr) * ROWB + (((2 * i + (mi & 1)) ^ swizzle<CH>(mr)) & mask) * 16;
  }
  uint32_t qf[KS][NQ][2];
  // m: the largest score; base: the same, 0 while it is -inf.  A weight is 2^((s - base) scale log2(e)): the distance first, which is
  // exact where it matters, so that scores of any size keep their weights (a product m scale log2(e) is off by 2^7 at 2^31)
  float o[KS][NQ][4], m[NQ][2], l[NQ][2], base[NQ][2];
  bool poison = false, fresh = true;
  int first_tile = cur.t, rows_here = 0, head0 = 0, slot = 0;
  while (left > 0) {
    if (fresh) {   // a new (request, head tile): its queries, empty statistics
      fresh = false;
      first_tile = cur.t;
      const int kvh = p.q_tiles == 1 ? cur.h : cur.h / p.q_tiles, qt = cur.h - kvh * p.q_tiles;
      head0 = kvh * p.group + qt * p.q_tile;
      rows_here = min(p.q_tile, p.group - qt * p.q_tile);
      const T* qb = static_cast<const T*>(p.q) + (int64_t)cur.b * p.q_sb + (int64_t)head0 * p.q_sh;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int r = n * 8 + g;
        const T* qr = qb + (int64_t)r * p.q_sh + t4 * 2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int d = ks * 16 + i * 8;
            qf[ks][n][i] = (r < rows_here && d < p.hd) ? (__ldg(reinterpret_cast<const uint32_t*>(qr + d)) ^ p.q_sign) & p.q_keep : 0u;
          }
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = base[n][0] = base[n][1] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) o[ks][n][0] = o[ks][n][1] = o[ks][n][2] = o[ks][n][3] = 0.f;
      }
      poison = false;
    }
    cp_async_wait<ST - 2>();
    __syncwarp();                       // the tile has come for every lane, and every lane is done with the slot before it
    issue(slot == 0 ? ST - 1 : slot - 1);
    look();
    poison |= (bad_bits >> slot) & 1u;
    const uint32_t tile = ring_u + slot * STAGE;

    // scores
    float s[MT][NQ][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t a[4];
        ldsm_x4(a, tile + kofs[ks & (NO - 1)] + (ks / 4) * 128 + i * 16 * ROWB);
#pragma unroll
        for (int n = 0; n < NQ; ++n) mma16816<T>(s[i][n], a[0], a[1], a[2], a[3], qf[ks][n][0], qf[ks][n][1]);
      }

    // running maximum and sum, in powers of two
    const int rows_in = cur.len - cur.t * TT;
    float mx[NQ][2];
    bool more = false;
    if (rows_in < TT) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if (i * 16 + g >= rows_in) s[i][n][0] = s[i][n][1] = -INFINITY;
          if (i * 16 + g + 8 >= rows_in) s[i][n][2] = s[i][n][3] = -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = m[n][e];
#pragma unroll
        for (int i = 0; i < MT; ++i) v = fmaxf(v, fmaxf(s[i][n][e], s[i][n][2 + e]));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        mx[n][e] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        more |= mx[n][e] > m[n][e];
      }
    }
    if (__any_sync(0xffffffffu, more)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float to = mx[n][e] == -INFINITY ? 0.f : mx[n][e];   // every score -inf so far: weights 0
          f[e] = m[n][e] == mx[n][e] ? 1.f : ex2((base[n][e] - to) * p.scale_log2);
          if (m[n][e] == -INFINITY) f[e] = 0.f;
          m[n][e] = mx[n][e];
          base[n][e] = to;
          l[n][e] *= f[e];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { o[ks][n][0] *= f[0]; o[ks][n][1] *= f[1]; o[ks][n][2] *= f[0]; o[ks][n][3] *= f[1]; }
      }
    }
    // output += weights * V; the weights go in as two summands so that their rounding stays below the output's
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      uint32_t hi[NQ][2], lo[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[i][n][e] = ex2(fmaf(s[i][n][e] - base[n][e], p.scale_log2, Raise<T>::kBits));
          s[i][n][2 + e] = ex2(fmaf(s[i][n][2 + e] - base[n][e], p.scale_log2, Raise<T>::kBits));
          l[n][e] += s[i][n][e] + s[i][n][2 + e];
        }
        split2<T>(s[i][n][0], s[i][n][1], hi[n][0], lo[n][0]);
        split2<T>(s[i][n][2], s[i][n][3], hi[n][1], lo[n][1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          hi[n][e] = movmatrix_trans(hi[n][e]);
          lo[n][e] = movmatrix_trans(lo[n][e]);
        }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4];
        ldsm_x4_trans(a, tile + vofs[ks & (NO - 1)] + (ks / 4) * 128 + i * 16 * ROWB);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          mma16816<T>(o[ks][n], a[0], a[1], a[2], a[3], hi[n][0], hi[n][1]);
          mma16816<T>(o[ks][n], a[0], a[1], a[2], a[3], lo[n][0], lo[n][1]);
        }
      }
    }
    slot = slot + 1 == ST ? 0 : slot + 1;
    --left;

    if (cur.t + 1 == cur.n || left == 0) {   // the pair's end, or the share's
      // It goes through shared memory into rows.  At the share's end to the ring's start, where it stays as a part for the CTA
      // to add up; else, eight rows at a time, through the slot just read (which is not filled again before the next tile) to
      // the workspace or, if the share held the whole pair, to the output.
      const bool whole = first_tile == 0 && cur.t + 1 == cur.n, stay = left == 0 && !whole;
      if (left == 0) cp_async_wait<0>();
      __syncwarp();
      float* so = reinterpret_cast<float*>(left == 0 ? ring : ring + (slot == 0 ? ST - 1 : slot - 1) * STAGE);
      float* po = stay ? so : p.part + ((int64_t)p.ctas * 2 + w) * p.part_floats;   // of a part
      T* ob = static_cast<T*>(p.out) + ((int64_t)cur.b * p.Hq + head0) * p.hd;
      const int ld = stay ? p.hd : p.hd + 4;                // (four more words per row: no bank conflicts)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float* rows_of = stay ? so + n * 8 * p.hd : so;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[n][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          l[n][e] = poison ? __int_as_float(0x7fc00000) : sum;
          const int r = n * 8 + t4 * 2 + e;
          if (r < rows_here) {
            const float f = whole ? 1.f / l[n][e] : 1.f;
            float* to = rows_of + (t4 * 2 + e) * ld + g;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (p.hd == HD || ks * 16 + i * 8 < p.hd) to[ks * 16 + i * 8] = o[ks][n][i * 2 + e] * f;
            if (g == 0) {
              if (!whole) *reinterpret_cast<float2*>(po + p.rows * p.hd + r * 2) = make_float2(m[n][e], l[n][e]);
              else if (p.lse) p.lse[(int64_t)cur.b * p.Hq + head0 + r] = log_sum<T>(m[n][e], l[n][e], p.scale_log2);
            }
          }
        }
        if (stay) continue;
        __syncwarp();
        const int here = min(8, rows_here - n * 8), per = whole ? p.hd / 8 : p.hd / 4;
        for (int u = lane; u < here * per; u += 32) {
          const int r = u / per;
          if (whole) {
            const int d = (u - r * per) * 8;
            const float4 x = *reinterpret_cast<const float4*>(so + r * ld + d), y = *reinterpret_cast<const float4*>(so + r * ld + d + 4);
            T eight[8] = {Cvt<T>::from_f(x.x), Cvt<T>::from_f(x.y), Cvt<T>::from_f(x.z), Cvt<T>::from_f(x.w),
                          Cvt<T>::from_f(y.x), Cvt<T>::from_f(y.y), Cvt<T>::from_f(y.z), Cvt<T>::from_f(y.w)};
            *reinterpret_cast<uint4*>(ob + (n * 8 + r) * p.hd + d) = *reinterpret_cast<const uint4*>(eight);
          } else {
            const int d = (u - r * per) * 4;
            *reinterpret_cast<float4*>(po + (n * 8 + r) * p.hd + d) = *reinterpret_cast<const float4*>(so + r * ld + d);
          }
        }
        __syncwarp();
      }
      if (!whole && lane == 0) {
        const int k = 2 * warp + (left == 0 ? 1 : 0);
        s_pair[k] = cur.b * H + cur.h;
        s_ends[k] = (first_tile == 0 ? 1 : 0) | (cur.t + 1 == cur.n ? 2 : 0);
      }
      __syncwarp();
      if (p.hd < HD && left > 0) {                          // the slot's padding chunks back to zero
        for (int u = lane; u < STAGE / 16; u += 32) reinterpret_cast<uint4*>(so)[u] = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      fresh = true;
    }
    if (left > 0) advance(cur);
  }
  // (a first part in the workspace comes back near the SM before the CTA adds it up)
  if (s_pair[2 * warp] >= 0)
    for (int i = lane * 32; i < p.part_floats; i += 1024) prefetch(p.part + ((int64_t)p.ctas * 2 + w) * p.part_floats + i);
  __syncthreads();

  // The parts of one pair, neighbours in the order of the warps' shares (place 2 w: warp w's first, in the workspace; 2 w + 1: its
  // last, in shared memory).  Several pairs are shared out over the warps.
  const int my_pair = lane < 2 * NW ? s_pair[lane] : -1;
  const unsigned same = __match_any_sync(0xffffffffu, my_pair);
  unsigned firsts = __ballot_sync(0xffffffffu, my_pair >= 0 && (same & ((1u << lane) - 1)) == 0);   // of each pair's parts
  const int quads = p.hd / 4, pairs = __popc(firsts);
  const int wpp = NW / max(1, min(pairs, NW));              // warps per pair
  for (int n = 0; n < pairs; ++n) {
    const int k0 = __ffs(firsts) - 1;
    firsts &= firsts - 1;
    const unsigned mask = __shfl_sync(0xffffffffu, same, k0);
    const int pair = __shfl_sync(0xffffffffu, my_pair, k0), ends = s_ends[k0] | s_ends[31 - __clz(mask)];
    if (n % (NW / wpp) != warp / wpp) continue;
    const int b = pair / H, h = pair - b * H;
    const int kvh = p.q_tiles == 1 ? h : h / p.q_tiles, qt = h - kvh * p.q_tiles;
    const int head = kvh * p.group + qt * p.q_tile, rows = min(p.q_tile, p.group - qt * p.q_tile);
    // (the join finds the part of a pair that began in a CTA before this one in place 0, of one that goes on in the next in 1)
    const int64_t t0 = (int64_t)s_cum[b] * H + (int64_t)h * (s_cum[b + 1] - s_cum[b]) + PC;   // the pair's first tile
    float* po = p.part + ((int64_t)blockIdx.x * 2 + (t0 < (int64_t)blockIdx.x * NW * share ? 0 : 1)) * p.part_floats;
    const float* in_ws = p.part + ((int64_t)p.ctas * 2 + blockIdx.x * NW) * p.part_floats;
    // (rolled up: this runs once, and what it costs is the way of its instructions to the SM)
#pragma unroll 1
    for (int i = (warp % wpp) * 32 + lane; i < rows * quads; i += wpp * 32) {
      const int r = i / quads, d = (i - r * quads) * 4;
      float m = -INFINITY, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (unsigned parts = mask; parts; parts &= parts - 1) {
        const int k = __ffs(parts) - 1;
        const float* part = (k & 1) ? reinterpret_cast<const float*>(smem + (k / 2) * ST * STAGE) : in_ws + (k / 2) * p.part_floats;
        const float2 ml = *reinterpret_cast<const float2*>(part + p.rows * p.hd + 2 * r);
        const float4 v = *reinterpret_cast<const float4*>(part + i * 4);
        const float to = fmaxf(m, ml.x), base = to == -INFINITY ? 0.f : to, f = ex2((m - base) * p.scale_log2), g = ex2((ml.x - base) * p.scale_log2);
        m = to;
        l = fmaf(l, f, g * ml.y);
        acc.x = fmaf(acc.x, f, g * v.x);
        acc.y = fmaf(acc.y, f, g * v.y);
        acc.z = fmaf(acc.z, f, g * v.z);
        acc.w = fmaf(acc.w, f, g * v.w);
      }
      if (ends == 3) {
        const float inv = 1.f / l;
        const int64_t at = (int64_t)b * p.Hq + head + r;
        T four[4] = {Cvt<T>::from_f(acc.x * inv), Cvt<T>::from_f(acc.y * inv), Cvt<T>::from_f(acc.z * inv), Cvt<T>::from_f(acc.w * inv)};
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * p.hd + d) = *reinterpret_cast<const uint2*>(four);
        if (d == 0 && p.lse) p.lse[at] = log_sum<T>(m, l, p.scale_log2);
      } else {
        *reinterpret_cast<float4*>(po + i * 4) = acc;
        if (d == 0) *reinterpret_cast<float2*>(po + p.rows * p.hd + 2 * r) = make_float2(m, l);
      }
    }
  }
}

// WPR warps per (request, query head): nothing where one share held the whole pair, zeros for an empty request, else the
// parts' weighted sum.  A warp takes every WPR-th part, its statistics one per lane, its values four side by side per lane.
template <typename T, int WPR>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p) {
  constexpr int RPC = 8 / WPR;                  // rows per CTA
  __shared__ __align__(16) float s_o[WPR > 1 ? WPR : 1][256];
  __shared__ float s_m[WPR], s_l[WPR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wi = warp % WPR;
  const int64_t rw = (int64_t)blockIdx.x * RPC + warp / WPR;   // WPR > 1: the same for the whole CTA
  const bool live = rw < (int64_t)p.B * p.Hq;
  const int b = live ? (int)(rw / p.Hq) : 0, hq = live ? (int)(rw - (int64_t)b * p.Hq) : 0;
  const int kvh = hq / p.group, in_group = hq - kvh * p.group, qt = in_group / p.q_tile, r = in_group - qt * p.q_tile;
  const int H = p.Hkv * p.q_tiles;
  T* ob = static_cast<T*>(p.out) + rw * p.hd;
  // The lengths are inputs, which the attention kernel's own start has waited for: a small batch is scanned before its end
  // (1 us of one request's 11).
  const bool early = p.B <= 256;
  int before = 0, all = 0, n = 0;
  if (early) {
    const int64_t cap = (int64_t)p.width * p.page_size;
    for (int a = lane; a < p.B; a += 32) {
      bool poison;
      const int len = clamp_len(__ldg(p.lens + a), cap, poison), t = len > 0 ? (len + p.tile - 1) / p.tile + p.pair_cost : 0;
      all += t;
      before += a < b ? t : 0;
      n += a == b ? t : 0;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, s);
      before += __shfl_xor_sync(0xffffffffu, before, s);
      n += __shfl_xor_sync(0xffffffffu, n, s);
    }
  } else {
    chain_wait();
    before = __ldcg(p.cum + b);
    n = __ldcg(p.cum + b + 1) - before;
    all = __ldcg(p.cum + p.B);
  }
  const int64_t total = (int64_t)all * H;
  const int64_t share = div_up(total, p.ctas * p.warps) * p.warps;             // of a CTA
  const int64_t t0 = (int64_t)before * H + (int64_t)(kvh * p.q_tiles + qt) * n + p.pair_cost, t1 = t0 + n - p.pair_cost;   // its tiles
  int w0 = 0, w1 = 0;
  if (n > 0) {
    w0 = total <= 0x7fffffff ? (int)((unsigned)t0 / (unsigned)share) : (int)(t0 / share);
    w1 = total <= 0x7fffffff ? (int)((unsigned)(t1 - 1) / (unsigned)share) : (int)((t1 - 1) / share);
  }
  const int64_t first = (int64_t)w0 * 2 + 1;     // (the part of the CTA that the pair begins in)
  const int parts = w1 - w0 + 1;
  if (early) chain_wait();
  if (!live) return;                            // (only with WPR = 1, where no barrier follows)
  if (n == 0) {   // an empty request; one with a length but no table at all is NaN like any that outgrew its table
    if (wi > 0) return;
    const bool wrong = p.lens[b] > 0;
    for (int d = lane; d < p.hd; d += 32) ob[d] = Cvt<T>::from_f(wrong ? __int_as_float(0x7fc00000) : 0.f);
    if (p.lse && lane == 0) p.lse[rw] = wrong ? __int_as_float(0x7fc00000) : -INFINITY;
    return;
  }
  if (parts == 1) return;
  auto at = [&](int i) { return p.part + (i == 0 ? first : (int64_t)(w0 + i) * 2) * p.part_floats; };
  const int d0 = lane * 4, d1 = d0 + 128;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
  float m = -INFINITY, l = 0.f;
  auto scaled = [](float4 x, float f, float4 y) { return make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w)); };
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = wi; i0 < parts; i0 += 32 * WPR) {
    const int mine = i0 + lane * WPR;           // this lane's part
    const float2 ml = mine < parts ? __ldcg(reinterpret_cast<const float2*>(at(mine) + p.rows * p.hd + 2 * r)) : make_float2(-INFINITY, 0.f);
    float mx = ml.x;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    mx = fmaxf(mx, m);
    const float base = mx == -INFINITY ? 0.f : mx, w = ex2((ml.x - base) * p.scale_log2);
    float sum = w * ml.y;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float f = m == -INFINITY ? 0.f : ex2((m - base) * p.scale_log2);
    l = fmaf(l, f, sum);
    m = mx;
    a = scaled(a, f, zero);
    c = scaled(c, f, zero);
    const int here = min(32, (parts - i0 + WPR - 1) / WPR);
#pragma unroll 8
    for (int k = 0; k < here; ++k) {
      const float f = __shfl_sync(0xffffffffu, w, k);
      const float* o = at(i0 + k * WPR) + r * p.hd;
      if (d0 < p.hd) a = scaled(__ldcg(reinterpret_cast<const float4*>(o + d0)), f, a);
      if (d1 < p.hd) c = scaled(__ldcg(reinterpret_cast<const float4*>(o + d1)), f, c);
    }
  }
  if constexpr (WPR > 1) {
    if (lane == 0) { s_m[wi] = m; s_l[wi] = l; }
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < WPR; ++w) all = fmaxf(all, s_m[w]);
    const float base = all == -INFINITY ? 0.f : all;
    const float f = ex2((m - base) * p.scale_log2);
    reinterpret_cast<float4*>(s_o[wi])[lane] = scaled(a, f, zero);
    if (p.hd > 128) reinterpret_cast<float4*>(s_o[wi])[lane + 32] = scaled(c, f, zero);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) l = fmaf(s_l[w], ex2((s_m[w] - base) * p.scale_log2), l);
    m = all;
    __syncthreads();
    const int d = threadIdx.x;
    if (d < p.hd) {
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) acc += s_o[w][d];
      ob[d] = Cvt<T>::from_f(acc / l);
    }
  } else {
    const float inv = 1.f / l;
    auto put = [&](int d, float4 v) {           // hd is a multiple of 8
      T four[4] = {Cvt<T>::from_f(v.x * inv), Cvt<T>::from_f(v.y * inv), Cvt<T>::from_f(v.z * inv), Cvt<T>::from_f(v.w * inv)};
      *reinterpret_cast<uint2*>(ob + d) = *reinterpret_cast<const uint2*>(four);
    };
    if (d0 < p.hd) put(d0, a);
    if (d1 < p.hd) put(d1, c);
  }
  if (p.lse && wi == 0 && lane == 0) p.lse[rw] = log_sum<T>(m, l, p.scale_log2);
}

int padded_hd(int hd) { return hd <= 16 ? 16 : (hd <= 32 ? 32 : (hd <= 64 ? 64 : (hd <= 128 ? 128 : 256))); }

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Heads per tile of a group: as few tiles as there can be, of one size.
int q_tile_for(int group, int HD) { return ceil_div(group, ceil_div(group, most_heads(HD))); }

int part_floats_of(int rows, int hd) { return ceil_div(rows * (hd + 2), 4) * 4; }   // 16-byte aligned parts

size_t workspace_for(int B, int Hq, int Hkv, int hd, int sms) {
  const int HD = padded_hd(hd), rows = q_tile_for(Hq / Hkv, HD);
  return round256((size_t)sms * (2 + warps_of(HD)) * part_floats_of(rows, hd) * 4) + round256(((size_t)B + 1) * 4);
}

template <typename T, int HD, int NQ>
int launch(const PagedParams& p, int sms, cudaStream_t st) {
  constexpr int NW = warps_of(HD);
  const size_t smem = (size_t)NW * stages_of(HD) * 2 * tile_tokens(HD) * HD * 2 + (size_t)(2 * p.B + 1) * 4;
  auto kern = p.page_size % 16 == 0 ? paged_attention_kernel<T, HD, NQ, true> : paged_attention_kernel<T, HD, NQ, false>;
  HB_PROPAGATE(ensure_dynamic_smem((const void*)kern, smem));
  kern<<<(unsigned)sms, NW * 32, smem, st>>>(p);
  HB_LAUNCH_CHECK();
  // a warp per row, or eight where a row has many parts (few pairs for the CTAs): one request of 1500 tokens takes 11.1 us with
  // eight and 14.0 with one, 64 requests 61.6 and 55.3
  const int64_t rows = (int64_t)p.B * p.Hq;
  if ((int64_t)p.B * p.Hkv * p.q_tiles * 4 <= sms) return launch_chained(paged_join_kernel<T, 8>, dim3((unsigned)rows), dim3(256), 0, st, true, 1, p);
  return launch_chained(paged_join_kernel<T, 1>, dim3((unsigned)ceil_div64(rows, 8)), dim3(256), 0, st, true, 1, p);
}

template <typename T, int NQ>
int launch_hd(const PagedParams& p, int sms, cudaStream_t st) {
  switch (padded_hd(p.hd)) {
    case 16: return launch<T, 16, NQ>(p, sms, st);
    case 32: return launch<T, 32, NQ>(p, sms, st);
    case 64: return launch<T, 64, NQ>(p, sms, st);
    case 128: return launch<T, 128, NQ>(p, sms, st);
    default: return launch<T, 256, 1>(p, sms, st);
  }
}

template <typename T>
int launch_group(const PagedParams& p, int sms, cudaStream_t st) {
  return p.rows <= 8 ? launch_hd<T, 1>(p, sms, st) : (p.rows <= 16 ? launch_hd<T, 2>(p, sms, st) : launch_hd<T, 3>(p, sms, st));
}

int check_heads(const char* what, int64_t B, int Hq, int Hkv, int hd) {
  HB_REQUIRE(B >= 0 && Hq >= 1 && Hkv >= 1 && hd >= 1, HB200_ERR_INVALID, "%s: bad shape B=%lld Hq=%d Hkv=%d hd=%d", what,
             (long long)B, Hq, Hkv, hd);
  HB_REQUIRE(Hq % Hkv == 0, HB200_ERR_INVALID, "%s: %d query heads are no multiple of %d kv heads", what, Hq, Hkv);
  HB_REQUIRE(hd % 8 == 0 && hd <= 256, HB200_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 256 is built)", what, hd);
  HB_REQUIRE(B <= kMaxBatch, HB200_ERR_UNSUPPORTED, "%s: %lld requests (up to %d in one call)", what, (long long)B, kMaxBatch);
  HB_REQUIRE(Hq <= 1024, HB200_ERR_UNSUPPORTED, "%s: %d query heads (up to 1024 are built)", what, Hq);
  return 0;
}

}  // namespace
}  // namespace hb200

using namespace hb200;

extern "C" size_t hb200_paged_attention_workspace_bytes(int B, int Hq, int Hkv, int hd) {
  int sms = 0;
  if (check_heads("paged_attention_workspace_bytes", B, Hq, Hkv, hd) != 0 || device_sms(&sms) != 0) return 0;
  return workspace_for(B, Hq, Hkv, hd, sms);
}

extern "C" int hb200_paged_decode_attention(const hb200_paged_cache* c, const void* q, int64_t q_stride_b, int64_t q_stride_h,
                                            void* out, float* lse, const int32_t* block_tables, int64_t table_ld, int table_width,
                                            const int32_t* kv_lens, int B, int Hq, float scale, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  HB_REQUIRE(c, HB200_ERR_INVALID, "paged_decode_attention: null pointer");
  HB_PROPAGATE(check_heads("paged_decode_attention", B, Hq, c->n_kv_heads, c->head_dim));
  if (B == 0) return 0;
  HB_REQUIRE(q && out && kv_lens && c->k && c->v && workspace, HB200_ERR_INVALID, "paged_decode_attention: null pointer");
  HB_REQUIRE(c->num_pages >= 0 && c->page_size >= 1 && table_width >= 0 && table_ld >= table_width && (block_tables || table_width == 0),
             HB200_ERR_INVALID, "paged_decode_attention: bad cache or table shape");
  HB_REQUIRE(aligned16(q) && aligned16(out) && aligned16(c->k) && aligned16(c->v) && aligned16(workspace), HB200_ERR_INVALID,
             "paged_decode_attention: pointers must be 16-byte aligned");
  const int64_t strides[] = {q_stride_b, q_stride_h, c->k_stride_page, c->k_stride_head, c->k_stride_row,
                             c->v_stride_page, c->v_stride_head, c->v_stride_row};
  for (int64_t s : strides)
    HB_REQUIRE(s % 8 == 0, HB200_ERR_INVALID, "paged_decode_attention: strides must be multiples of 8 elements");
  HB_REQUIRE(scale - scale == 0.f, HB200_ERR_INVALID, "paged_decode_attention: scale is NaN or infinite");
  // lengths are clamped to the table's reach, so this bounds every tile count in 32 bits
  const int64_t cap = (int64_t)table_width * c->page_size;
  HB_REQUIRE(cap <= 0x7fffff00 && (int64_t)B * (cap / 16 + 4) <= 0x7fffffff, HB200_ERR_UNSUPPORTED,
             "paged_decode_attention: tables of %d pages of %d tokens for %d requests reach too far", table_width, c->page_size, B);
  HB_REQUIRE((cap / 16 + 4) * Hq <= 0x7fffffff, HB200_ERR_UNSUPPORTED,
             "paged_decode_attention: tables of %d pages of %d tokens for %d query heads reach too far", table_width, c->page_size, Hq);
  // Warps store what they have finished while others still read.
  const Reach k_reach = reach_of(c->k, c->head_dim * 2, {{c->num_pages, c->k_stride_page * 2}, {c->n_kv_heads, c->k_stride_head * 2}, {c->page_size, c->k_stride_row * 2}});
  const Reach v_reach = reach_of(c->v, c->head_dim * 2, {{c->num_pages, c->v_stride_page * 2}, {c->n_kv_heads, c->v_stride_head * 2}, {c->page_size, c->v_stride_row * 2}});
  const Reach read[] = {reach_of(q, c->head_dim * 2, {{B, q_stride_b * 2}, {Hq, q_stride_h * 2}}), k_reach, v_reach,
                        reach_of(block_tables, (int64_t)table_width * 4, {{B, table_ld * 4}}), reach_of(kv_lens, (int64_t)B * 4)};
  const Reach written[] = {reach_of(out, (int64_t)B * Hq * c->head_dim * 2), reach_of(lse, lse ? (int64_t)B * Hq * 4 : 0)};
  for (const Reach& w : written)
    for (const Reach& r : read)
      HB_REQUIRE(!overlap(w, r), HB200_ERR_INVALID, "paged_decode_attention: out and lse must not overlap what is read");
  HB_REQUIRE(!overlap(written[0], written[1]), HB200_ERR_INVALID, "paged_decode_attention: out and lse must not overlap one another");
  const int group = Hq / c->n_kv_heads;
  int sms = 0;
  HB_PROPAGATE(device_sms(&sms));
  HB_REQUIRE(workspace_bytes >= workspace_for(B, Hq, c->n_kv_heads, c->head_dim, sms), HB200_ERR_WORKSPACE,
             "paged_decode_attention: workspace of %zu bytes, needs %zu", workspace_bytes,
             workspace_for(B, Hq, c->n_kv_heads, c->head_dim, sms));
  PagedParams p = {};
  p.q = q; p.kc = c->k; p.vc = c->v; p.out = out; p.lse = lse; p.table = block_tables; p.lens = kv_lens;
  p.q_sb = q_stride_b; p.q_sh = q_stride_h;
  p.k_sh = c->k_stride_head; p.v_sh = c->v_stride_head;
  const int64_t in_bytes[] = {c->k_stride_page * 2, c->k_stride_row * 2, c->v_stride_page * 2, c->v_stride_row * 2};
  for (int64_t x : in_bytes)
    HB_REQUIRE(x >= -0x7fffffffll && x <= 0x7fffffffll, HB200_ERR_UNSUPPORTED, "paged_decode_attention: pages or rows more than 2 GB apart");
  p.k_sp = (int32_t)in_bytes[0]; p.k_sr = (int32_t)in_bytes[1]; p.v_sp = (int32_t)in_bytes[2]; p.v_sr = (int32_t)in_bytes[3];
  p.table_ld = table_ld;
  p.B = B; p.Hq = Hq; p.Hkv = c->n_kv_heads; p.hd = c->head_dim; p.group = group;
  const int HD = padded_hd(c->head_dim);
  p.q_tile = p.rows = q_tile_for(group, HD);
  p.q_tiles = ceil_div(group, p.q_tile);
  p.part_floats = part_floats_of(p.rows, p.hd);
  p.tile = tile_tokens(HD);
  p.pair_cost = pair_cost(HD);
  p.warps = warps_of(HD);
  p.page_size = c->page_size; p.width = table_width; p.num_pages = c->num_pages;
  p.ctas = sms;
  // (from the smallest scale to the largest it stays above zero and finite, for distances of zero and of infinity)
  const double log2_scale = (scale < 0.f ? -(double)scale : (double)scale) * 1.4426950408889634;
  p.scale_log2 = scale == 0.f ? 1.f : (log2_scale < FLT_MAX ? (float)log2_scale : FLT_MAX);
  p.q_keep = scale == 0.f ? 0u : 0xffffffffu;
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.cum = reinterpret_cast<int32_t*>(ws + round256((size_t)sms * (2 + p.warps) * p.part_floats * 4));
  cudaStream_t st = (cudaStream_t)stream;
  if (c->dtype == HB200_BF16) return launch_group<__nv_bfloat16>(p, sms, st);
  if (c->dtype == HB200_F16) return launch_group<__half>(p, sms, st);
  set_error("paged_decode_attention: unsupported dtype %d (bf16 and f16 are built)", c->dtype);
  return HB200_ERR_UNSUPPORTED;
}
