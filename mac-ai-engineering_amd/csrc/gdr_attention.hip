// Attention over a paged 4-bit cache (gdr_kv4.h has its format), for MI355X (gfx950):
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i k_j - m_i),   j <= the position of query i
//
// over any number of requests at once: request r has `len` tokens in the cache, the last of which are its queries (one
// when a token is generated, several when drafts are checked, a chunk of a prompt).  G = Hq / Hk query heads share a key
// head; a request's queries and the G heads of each are G qlen rows that read the same keys, taken R at a time.
//
// One pass over the keys with the running maximum and sum of the softmax, in 32 bits, on the matrix cores: S^T = K Q^T and
// O^T = V^T P^T, both v_mfma_f32_16x16x32_bf16 on operands that stay in registers.  Keys and values are decoded to bf16,
// which holds them exactly (2 bits of mantissa, a power of two), so a bf16 query loses nothing on the way in; P is rounded
// to bf16 once (at most 2^-8 of it, as the output is).  float16 and float32 queries, and their P, are the sum of two bf16
// terms each (at most 2^-16 off), at twice the products: the decoded operands are the same.
//   - S^T's accumulator (lane 16 h + n: query row n, tokens 4 h + i) is P^T's operand for 32 tokens in the order 4 h + 0..3,
//     16 + 4 h + 0..3; the values are stored so that the same lane loads those tokens.  No exchange of P, no transposition.
//   - O^T's columns are query rows, so a row's maximum, sum and rescaling are one lane's scalars.
//   - The reference maximum moves only when some row's scores pass it by 2^8 (P stays below 2^8, far from any limit):
//     most steps need no reduction over lanes and no rescaling.
//
// Work is split evenly over the chip, whatever the lengths are: all requests' keys, times heads, times groups of rows, are
// one line of tokens, and each workgroup takes an equal stretch of it, found from the lengths on the device.  A stretch
// that covers part of a row group leaves its m, sum and O (32 bits) in the workspace, and a second launch joins them.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gdr_abi.h"
#include "gdr_common.h"
#include "gdr_kv4.h"

namespace gdr {

typedef _Float16 f16;
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned long long u64;

constexpr int AT_WAVES = 4;
constexpr float AT_LOWEST = -3.402823466e38f;    // a reference maximum below every score; exp2(-inf - it) is 0
constexpr float AT_SLACK = 8.f;                  // how far (log2) scores may pass the reference maximum

struct AttnArgs {
  const void* q;
  void* o;
  const uint8_t* cache;
  const int *blocks, *lens, *starts;             // starts null: request r's one query is row r
  float* part;                                   // [2 workers][R rows][D + 2]: O, then m and the sum
  int4* records;                                 // [workers]: {request, head and row group, last worker, 1 if any}
  int64_t q_row, q_head;                         // strides in elements
  int64_t T, B, W, pages;
  int Hq, Hk, page, page_shift, workers;
  float scale;                                   // times log2 e
};

// A request as the split sees it.  Costs are in tokens: a row group j of a head costs base + (j + 1) per, the keys its
// last row sees, rounded up where G does not divide R (a few tokens too many, never too few).
struct Req {
  int q0, qlen, len, base;                       // first query row, queries, tokens, tokens before the queries
  int groups;                                    // row groups a head
  __device__ __forceinline__ int64_t cost(int64_t j, int per) const { return j * base + (int64_t)per * j * (j + 1) / 2; }
};

template <int R>
__device__ __forceinline__ Req request(const AttnArgs& a, int64_t r, int G) {
  Req x;
  const int64_t most = a.W * a.page;
  x.len = (int)min((int64_t)max(a.lens[r], 0), most);
  if (a.starts) {
    x.q0 = (int)min((int64_t)max(a.starts[r], 0), a.T);
    x.qlen = (int)min((int64_t)max(a.starts[r + 1] - x.q0, 0), a.T - x.q0);
  } else {
    x.q0 = (int)r;
    x.qlen = 1;
  }
  x.base = max(x.len - x.qlen, 0);
  x.groups = (int)(((int64_t)x.qlen * G + R - 1) / R);
  return x;
}

__device__ __forceinline__ int64_t uniform(int64_t x) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)x);
  const unsigned hi = __builtin_amdgcn_readfirstlane((int)(unsigned)((u64)x >> 32));
  return (int64_t)((u64)hi << 32 | lo);
}

// floor(x / y), 0 <= x < 2^53, 0 < y < 2^53
__device__ __forceinline__ int64_t div64(int64_t x, int64_t y) {
  int64_t q = (int64_t)((double)x / (double)y);
  if (q * y > x) --q;
  if ((q + 1) * y <= x) ++q;
  return q;
}

// ---- where a workgroup's stretch begins -----------------------------------------------------------------------------
struct Place {
  int64_t share, total, r, before;               // cost before request r
};

// The stretch's length and the request at offset `w * share` of the line (r = B past its end).  All requests' costs are
// summed by the whole workgroup, 256 at a time.
template <int R>
__device__ __forceinline__ Place find(const AttnArgs& a, int w, int G, int per, int step) {
  __shared__ int64_t sums[AT_WAVES];
  __shared__ int64_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Place p;
  p.total = 0;
  int64_t mine = 0, incl = 0;                    // of the last 256 requests, kept for the second pass
  const int64_t rounds = (a.B + 255) / 256;
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t r = i * 256 + tid;
    mine = 0;
    if (r < a.B) {
      const Req x = request<R>(a, r, G);
      mine = x.cost(x.groups, per) * a.Hk;
    }
    incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t y = __shfl_up(incl, d);
      if (lane >= d) incl += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < AT_WAVES; ++v) p.total += sums[v];
  }
  p.share = div64(p.total + a.workers - 1, a.workers);
  p.share = max((p.share + step - 1) / step * step, (int64_t)step);
  const int64_t at = p.share * w;
  if (tid == 0) found[0] = a.B, found[1] = 0;
  __syncthreads();
  if (at < p.total) {
    int64_t before = 0;
    for (int64_t i = 0; i < rounds; ++i) {
      const int64_t r = i * 256 + tid;
      if (rounds > 1) {
        mine = 0;
        if (r < a.B) {
          const Req x = request<R>(a, r, G);
          mine = x.cost(x.groups, per) * a.Hk;
        }
        incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int64_t y = __shfl_up(incl, d);
          if (lane >= d) incl += y;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = incl;
        __syncthreads();
      }
      int64_t b = before + incl - mine;
#pragma unroll
      for (int v = 0; v < AT_WAVES; ++v) {
        if (v < wave) b += sums[v];
        before += sums[v];
      }
      if (at >= b && at < b + mine) found[0] = r, found[1] = b;   // one thread of all
    }
    __syncthreads();
  }
  p.share = uniform(p.share);
  p.total = uniform(p.total);
  p.r = uniform(found[0]);
  p.before = uniform(found[1]);
  return p;
}

// ---- a wave's part -----------------------------------------------------------------------------------------------
template <int D>
struct Tile {                                    // 32 tokens' codes and scales as loaded
  static constexpr int NC = D < 128 ? 1 : D / 128, NW = D < 128 ? 2 : 4;
  unsigned kc[2][NC][NW], vc[2][NC][NW], ks[2][NC], vs[2][NC];
};

template <int D>
__device__ __forceinline__ void load_sub(const uint8_t* k, const uint8_t* v, Tile<D>& t, int s, int lane) {
  using TT = Tile<D>;
  const int h = lane >> 4, m = lane & 15;
  if constexpr (D == 64) {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(k + (h >> 1) * 256 + m * 16 + (h & 1) * 8);
    const u32x2_t y = *reinterpret_cast<const u32x2_t*>(v + lane * 8);
    t.kc[s][0][0] = x[0], t.kc[s][0][1] = x[1];
    t.vc[s][0][0] = y[0], t.vc[s][0][1] = y[1];
    t.ks[s][0] = k[8 * D + (h >> 1) * 16 + m];
    t.vs[s][0] = *reinterpret_cast<const unsigned*>(v + 8 * D + h * (D / 8) + (m >> 3) * 4);
  } else {
#pragma unroll
    for (int c = 0; c < TT::NC; ++c) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(k + c * 1024 + lane * 16);
      const u32x4_t y = *reinterpret_cast<const u32x4_t*>(v + c * 1024 + lane * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) t.kc[s][c][i] = x[i], t.vc[s][c][i] = y[i];
      t.ks[s][c] = k[8 * D + c * 64 + lane];
      t.vs[s][c] = *reinterpret_cast<const unsigned*>(v + 8 * D + h * (D / 8) + (4 * c + (m >> 2)) * 4);
    }
  }
}

// 8 codes as a bf16 operand fragment.
__device__ __forceinline__ bf16x8 decode8(unsigned w, float s) {
  return __builtin_bit_cast(bf16x8, u32x4_t{kv_decode2<0>(w, s), kv_decode2<1>(w, s), kv_decode2<2>(w, s),
                                            kv_decode2<3>(w, s)});
}

template <typename T>
__device__ __forceinline__ void load_f8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f4 a = *reinterpret_cast<const f4*>(p), b = *reinterpret_cast<const f4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = *reinterpret_cast<const T8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  }
}

// NQ blocks of 16 query rows of a wave: their operands, O^T, reference maxima and sums.
template <typename T, int D, int NQ>
struct Rows {
  static constexpr int TERMS = sizeof(T) == 2 && std::is_same<T, bf16>::value ? 1 : 2;
  static constexpr int STEPS = D / 32, ND = D / 16;
  bf16x8 q[NQ][TERMS][STEPS];
  f4 o[NQ][ND];
  float m[NQ], l[NQ];
  int last[NQ];                                  // the last key the lane's row sees; -1: a row that does not exist

  // row0: the first of the wave's rows within the request and head
  __device__ __forceinline__ void begin(const AttnArgs& a, const Req& x, int head, int row0, int G, int lane) {
    const int h = lane >> 4, n = lane & 15;
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      const int row = row0 + b * 16 + n, i = row / G, g = row - i * G;
      const bool there = i < x.qlen;
      last[b] = there ? x.len - x.qlen + i : -1;
      const T* p = (const T*)a.q + (x.q0 + (there ? i : 0)) * a.q_row + (int64_t)(head * G + g) * a.q_head;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        // the channels of a key that lane quarter h holds in step s
        const int ch = D == 64 ? h * 16 + s * 8 : (s / 4 * 4 + h) * 32 + s % 4 * 8;
        float v[8];
        load_f8(p + ch, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = there ? v[e] : 0.f;
          const bf16 hi = (bf16)f;
          q[b][0][s][e] = hi;
          if constexpr (TERMS == 2) q[b][1][s][e] = (bf16)(f - (float)hi);
        }
      }
#pragma unroll
      for (int t = 0; t < ND; ++t) o[b][t] = f4{0.f, 0.f, 0.f, 0.f};
      m[b] = AT_LOWEST;
      l[b] = 0.f;
    }
  }

  // 32 tokens from key t0 on.  MASKED: some row may not see all of them (their keys are masked, and values past kend,
  // which may be anything, are cleared).  P is two terms there: a row of few keys, whose keys are all in such tiles, does
  // not average the roundings of one.
  template <bool MASKED>
  __device__ __forceinline__ void step(Tile<D>& t, int t0, int kend, float scale, int lane) {
    using TT = Tile<D>;
    constexpr int PT = MASKED ? 2 : TERMS;
    const int h = lane >> 4;
    f4 s[NQ][2];
#pragma unroll
    for (int b = 0; b < NQ; ++b) s[b][0] = s[b][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < TT::NC; ++c) {
        const float ks = kv_scale(t.ks[u][c]);
#pragma unroll
        for (int i = 0; i < TT::NW; ++i) {
          const bf16x8 k = decode8(t.kc[u][c][i], ks);
#pragma unroll
          for (int b = 0; b < NQ; ++b)
#pragma unroll
            for (int w = 0; w < TERMS; ++w)
              s[b][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[b][w][c * 4 + i], s[b][u], 0, 0, 0);
        }
      }
    unsigned nan[NQ][TT::NC];                    // MASKED: the groups of a row's values that read as NaN
    if constexpr (MASKED) hide(t, s, nan, t0, kend, h);
    bf16x8 p[NQ][PT];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      float top = fmaxf(fmaxf(fmaxf(s[b][0][0], s[b][0][1]), fmaxf(s[b][0][2], s[b][0][3])),
                        fmaxf(fmaxf(s[b][1][0], s[b][1][1]), fmaxf(s[b][1][2], s[b][1][3]))) * scale;
      if (__any(top > m[b] + AT_SLACK)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m[b]);
        const float f = __builtin_amdgcn_exp2f(m[b] - top);
        m[b] = top;
        l[b] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[b][d] *= f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][u][i], scale, -m[b]));
          l[b] += e;
          const bf16 hi = (bf16)e;
          p[b][0][4 * u + i] = hi;
          if constexpr (PT == 2) p[b][1][4 * u + i] = (bf16)(e - (float)hi);
        }
    }
    values(t, p);
    if constexpr (MASKED) {
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int d = 0; d < ND; ++d)             // the lane's channels of a chunk are one group's
          if (nan[b][d / (ND / TT::NC)] >> (D == 64 ? h / 2 * 8 : 4 * h) & 1u) o[b][d] = f4(__builtin_nanf(""));
    }
  }

  // Masks the keys that rows do not see and clears the values past kend and those that read as NaN (0 times NaN is not 0:
  // a NaN goes to the rows that see it by itself).  nan: bit m of [b][c] is set where the row sees a NaN in the group that
  // lanes m load of chunk c.
  __device__ __forceinline__ void hide(Tile<D>& t, f4 (&s)[NQ][2], unsigned (&nan)[NQ][Tile<D>::NC], int t0, int kend, int h) {
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int c = 0; c < Tile<D>::NC; ++c) nan[b][c] = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = t0 + 16 * u + i, mine = at + 4 * h;
#pragma unroll
        for (int b = 0; b < NQ; ++b) s[b][u][i] = mine <= last[b] ? s[b][u][i] : -__builtin_inff();
#pragma unroll
        for (int c = 0; c < Tile<D>::NC; ++c) {
          const bool bad = mine < kend && (t.vs[u][c] >> (8 * i) & 0xFFu) == 0xFFu;
          const u64 lanes = __ballot(bad);
          if (lanes) {
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
              for (int v = 0; v < 4; ++v)
                if (at + 4 * v <= last[b]) nan[b][c] |= (unsigned)(lanes >> (16 * v)) & 0xFFFFu;
          }
          if (bad || mine >= kend) {
            if constexpr (D == 64) t.vc[u][c][i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
            else t.vc[u][c][i] = 0;
            t.vs[u][c] &= ~(0xFFu << (8 * i));
          }
        }
      }
  }

  // O^T += V^T P^T for the tile's 32 tokens.
  template <int PT>
  __device__ __forceinline__ void values(const Tile<D>& t, const bf16x8 (&p)[NQ][PT]) {
    constexpr int PER = ND / Tile<D>::NC;
    two_tiles<0>(t, p);
    if constexpr (PER > 2) two_tiles<1>(t, p);
    if constexpr (PER > 4) {
      two_tiles<2>(t, p);
      two_tiles<3>(t, p);
    }
  }

  // Byte SEL of every token's codes: the lane's channels 2 SEL and 2 SEL + 1 of each run, one output tile each.
  template <int SEL, int PT>
  __device__ __forceinline__ void two_tiles(const Tile<D>& t, const bf16x8 (&p)[NQ][PT]) {
    using TT = Tile<D>;
#pragma unroll
    for (int c = 0; c < TT::NC; ++c) {
      unsigned x[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned sc = t.vs[u][c];
        if constexpr (D == 64) {                 // a token's two bytes: tokens 0, 1 in the first word, 2, 3 in the second
          x[4 * u + 0] = kv_decode2<SEL>(t.vc[u][c][0], kv_scale(sc & 0xFFu));
          x[4 * u + 1] = kv_decode2<SEL + 2>(t.vc[u][c][0], kv_scale(sc >> 8 & 0xFFu));
          x[4 * u + 2] = kv_decode2<SEL>(t.vc[u][c][1], kv_scale(sc >> 16 & 0xFFu));
          x[4 * u + 3] = kv_decode2<SEL + 2>(t.vc[u][c][1], kv_scale(sc >> 24));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[4 * u + i] = kv_decode2<SEL>(t.vc[u][c][i], kv_scale(sc >> (8 * i) & 0xFFu));
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], half ? 0x07060302u : 0x05040100u);
        const bf16x8 v = __builtin_bit_cast(bf16x8, w);
        const int d = c * (ND / TT::NC) + 2 * SEL + half;
#pragma unroll
        for (int b = 0; b < NQ; ++b)
#pragma unroll
          for (int k = 0; k < PT; ++k) o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[b][k], o[b][d], 0, 0, 0);
      }
    }
  }

  // The rows' sums over the lanes that share them.
  __device__ __forceinline__ void end() {
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      l[b] += __shfl_xor(l[b], 16);
      l[b] += __shfl_xor(l[b], 32);
    }
  }
};

// Where lane 16 h + n's element i of output tile d is among a head's channels.
template <int D>
__device__ __forceinline__ int channel(int d, int h, int i) {
  constexpr int RUN = D < 128 ? D / 16 : 8;      // channels of a lane's run, and tiles of a chunk of 16 RUN channels
  return d / RUN * (16 * RUN) + (4 * h + i) * RUN + d % RUN;
}

// Waves a SIMD holds of the kernel that streams keys for 16 rows: what keeps enough loads in flight (a tile a wave) and
// fits the registers.
constexpr int waves_for(int D) { return D == 256 ? 2 : D == 128 ? 3 : 4; }

// KEYS: the workgroup's waves take different keys of the same 16 NQ rows and join their results at the end (few rows);
// else different rows of the same keys (16 NQ each).
template <typename T, int D, int NQ, bool KEYS>
__global__ void __launch_bounds__(64 * AT_WAVES, KEYS && NQ == 1 ? waves_for(D) : 1) attend_kernel(AttnArgs a) {
  using RT = Rows<T, D, NQ>;
  constexpr int R = 16 * NQ * (KEYS ? 1 : AT_WAVES), STEP = KEYS ? 32 * AT_WAVES : 32, ND = RT::ND;
  constexpr int RUN = D < 128 ? D / 16 : 8;
  __shared__ f4 join_o[KEYS ? 2 : 1][KEYS ? NQ * ND : 1][64];
  __shared__ float join_m[KEYS ? AT_WAVES : 1][NQ][16], join_l[KEYS ? AT_WAVES : 1][NQ][16];
  const int lane = threadIdx.x & 63, h = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.Hq / a.Hk, per = (R + G - 1) / G;
  const int w = blockIdx.x;
  const Place at = find<R>(a, w, G, per, STEP);
  int4 record = {0, 0, 0, 0};
  if (a.starts) {                                // query rows past the last request's have nothing to attend to
    const int64_t used = min((int64_t)max(a.starts[a.B], 0), a.T);
    for (int64_t t = used + w; t < a.T; t += a.workers)
      for (int i = threadIdx.x; i < a.Hq * D; i += 64 * AT_WAVES) ((T*)a.o)[t * a.Hq * D + i] = (T)0.f;
  }
  int64_t x0 = at.share * w;
  const int64_t x1 = min(x0 + at.share, at.total);
  int64_t before = at.before;
  bool opening = true;                           // the stretch's first piece: it may have begun in another
  for (int64_t r = at.r; r < a.B && x0 < x1;) {
    const Req x = request<R>(a, r, G);
    const int64_t each = x.cost(x.groups, per);  // of a head
    if (x0 >= before + each * a.Hk) {
      before += each * a.Hk;
      ++r;
      continue;
    }
    const int head = (int)uniform(div64(x0 - before, each));
    const int64_t y = x0 - before - head * each;
    int j = 0;
    for (int lo = 0, hi = x.groups - 1;; ) {     // the row group at y
      if (lo >= hi) { j = lo; break; }
      const int mid = (lo + hi + 1) / 2;
      if (x.cost(mid, per) <= y) lo = mid;
      else hi = mid - 1;
    }
    const int64_t u0 = before + head * each + x.cost(j, per), u1 = before + head * each + x.cost(j + 1, per);
    const int64_t stop = min(u1, x1);
    // the keys: the last row's at the most, both ends of a split rounded to whole steps
    const int rows = min(R, x.qlen * G - j * R), kall = x.len - x.qlen + (j * R + rows - 1) / G + 1;
    const int kmin = x.len - x.qlen + (j * R) / G + 1;          // keys that every row sees
    int ka = (int)(x0 - u0) / STEP * STEP, kb = stop == u1 ? kall : (int)(stop - u0) / STEP * STEP;
    kb = min(kb, kall);

    RT rw;
    rw.begin(a, x, head, j * R + (KEYS ? 0 : wave * 16 * NQ), G, lane);
    // A wave's tiles, the next one's loads in flight while one is worked on, and the page numbers a tile before those.
    const int* table = a.blocks + r * a.W;
    const int64_t pb = kv_page_bytes(a.page, D);
    const uint8_t* base = a.cache + (int64_t)head * pb;
    bool bad = false;
    int ids[2];
    const auto look = [&](int t0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) ids[u] = table[min(t0 + 16 * u, kb - 1) >> a.page_shift];
    };
    const auto fetch = [&](int t0, Tile<D>& tile) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool ok = (unsigned)ids[u] < (unsigned)a.pages;
        bad |= !ok;
        const uint8_t* k = base + (ok ? ids[u] : 0) * (2 * a.Hk * pb) +
                           ((t0 + 16 * u) & (a.page - 1)) / KV_SUB * kv_sub_bytes(D);
        load_sub<D>(k, k + a.Hk * pb, tile, u, lane);
      }
    };
    const int full = min(kmin, kb);
    int t0 = ka + (KEYS ? 32 * wave : 0);
    Tile<D> tile;
    if (t0 < kb) {
      look(t0);
      fetch(t0, tile);
      look(t0 + STEP);
    }
    while (t0 + 32 <= full) {
      Tile<D> next;
      fetch(t0 + STEP, next);
      look(t0 + 2 * STEP);
      rw.template step<false>(tile, t0, kb, a.scale, lane);
      tile = next;
      t0 += STEP;
    }
    while (t0 < kb) {
      rw.template step<true>(tile, t0, kb, a.scale, lane);
      t0 += STEP;
      fetch(t0, tile);
      look(t0 + STEP);
    }
    rw.end();
    if constexpr (KEYS) {                        // join the waves: 2, 3 into 0, 1, then 1 into 0
      __syncthreads();                           // the piece before has been read
#pragma unroll
      for (int b = 0; b < NQ; ++b)
        if (h == 0) join_m[wave][b][n] = bad ? __builtin_nanf("") : rw.m[b], join_l[wave][b][n] = rw.l[b];
      __syncthreads();
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        float m = AT_LOWEST, l = 0.f;
        bool poison = false;
        for (int v = 0; v < AT_WAVES; ++v) {
          poison |= __isnanf(join_m[v][b][n]);
          m = fmaxf(m, join_m[v][b][n]);
        }
        for (int v = 0; v < AT_WAVES; ++v) l += join_l[v][b][n] * __builtin_amdgcn_exp2f(join_m[v][b][n] - m);
        const float f = __builtin_amdgcn_exp2f(rw.m[b] - m);
        rw.m[b] = m;
        rw.l[b] = poison ? __builtin_nanf("") : l;
#pragma unroll
        for (int d = 0; d < ND; ++d) rw.o[b][d] *= f;
      }
#pragma unroll
      for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
          for (int b = 0; b < NQ; ++b)
#pragma unroll
            for (int d = 0; d < ND; ++d) join_o[wave - half][b * ND + d][lane] = rw.o[b][d];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
          for (int b = 0; b < NQ; ++b)
#pragma unroll
            for (int d = 0; d < ND; ++d) rw.o[b][d] += join_o[wave][b * ND + d][lane];
        }
        __syncthreads();
      }
    } else if (bad) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) rw.l[b] = __builtin_nanf("");
    }
    const bool whole = x0 == u0 && stop == u1;
    if (!KEYS || wave == 0) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const int lrow = (KEYS ? 0 : wave * 16 * NQ) + b * 16 + n, row = j * R + lrow, i = row / G, g = row - i * G;
        if (whole) {
          if (i >= x.qlen) continue;
          const float inv = rw.l[b] == 0.f ? 0.f : 1.f / rw.l[b];
          T* p = (T*)a.o + ((int64_t)(x.q0 + i) * a.Hq + head * G + g) * D;
#pragma unroll
          for (int c = 0; c < ND / RUN; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              typedef T TR __attribute__((ext_vector_type(RUN)));
              TR v;
#pragma unroll
              for (int f = 0; f < RUN; ++f) v[f] = (T)(rw.o[b][c * RUN + f][e] * inv);
              *reinterpret_cast<TR*>(p + channel<D>(c * RUN, h, e)) = v;
            }
        } else {
          float* p = a.part + ((int64_t)(2 * w + (opening ? 0 : 1)) * R + lrow) * (D + 4);
#pragma unroll
          for (int c = 0; c < ND / RUN; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int f = 0; f < RUN; f += 4)
                *reinterpret_cast<f4*>(p + channel<D>(c * RUN, h, e) + f) =
                    f4{rw.o[b][c * RUN + f][e], rw.o[b][c * RUN + f + 1][e], rw.o[b][c * RUN + f + 2][e],
                       rw.o[b][c * RUN + f + 3][e]};
          if (h == 0) p[D] = rw.m[b], p[D + 1] = rw.l[b];
        }
      }
    }
    if (x0 == u0 && stop != u1)                  // this workgroup begins a row group that others go on with
      record = {(int)r, head * x.groups + j, (int)div64(u1 - 1, at.share), opening ? 1 : 2};
    opening = false;
    x0 = stop;
  }
  if (threadIdx.x == 0) a.records[w] = record;
}

// Joins the parts of each row group that several workgroups worked on: block (w, y) the rows 4 y .. 4 y + 3 of the one that
// workgroup w began, a wave a row.
template <typename T, int D, int R>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a) {
  const int w = blockIdx.x, lane = threadIdx.x & 63, lrow = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int4 rec = a.records[w];
  if (!rec.w) return;
  const int G = a.Hq / a.Hk;
  const Req x = request<R>(a, rec.x, G);
  const int head = rec.y / x.groups, j = rec.y - head * x.groups;
  const int row = j * R + lrow, i = row / G, g = row - i * G;
  if (i >= x.qlen) return;
  constexpr int PER = D / 64;
  const auto at = [&](int v) { return a.part + ((int64_t)(2 * v + (v == w ? rec.w - 1 : 0)) * R + lrow) * (D + 4); };
  float m = AT_LOWEST, l = 0.f, o[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.f;
  for (int v = w; v <= rec.z; ++v) {
    const float* p = at(v);
    const float pm = p[D], pl = p[D + 1], top = fmaxf(m, pm);
    const float f = __builtin_amdgcn_exp2f(m - top), g2 = __builtin_amdgcn_exp2f(pm - top);
    m = top;
    l = l * f + pl * g2;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = o[e] * f + p[lane * PER + e] * g2;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* p = (T*)a.o + ((int64_t)(x.q0 + i) * a.Hq + head * G + g) * D + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) p[e] = (T)(o[e] * inv);
}

// ---- launches ---------------------------------------------------------------------------------------------------------
// Rows a wave takes and how the waves share the work, by the rows a request has on average: up to 16, and up to 32, the
// waves split the keys (the chip is filled by keys alone); above, the rows.
struct Shape {
  int nq;
  bool keys;
  int rows() const { return 16 * nq * (keys ? 1 : AT_WAVES); }
};
static Shape shape_for(int64_t T, int64_t B, int64_t G) {
  const int64_t rows = (T + B - 1) / B * G;
  if (rows <= 16) return {1, true};
  if (rows <= 32) return {2, true};
  return {2, false};
}
static int workers_for(const Shape& s, int64_t D) { return 256 * (s.keys && s.nq == 1 ? waves_for((int)D) : 1); }

template <typename T, int D>
static void launch(const Shape& s, const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.workers), join((unsigned)a.workers, (unsigned)(s.rows() / 4));
  if (s.keys && s.nq == 1) {
    hipLaunchKernelGGL((attend_kernel<T, D, 1, true>), grid, dim3(64 * AT_WAVES), 0, st, a);
    hipLaunchKernelGGL((join_kernel<T, D, 16>), join, dim3(256), 0, st, a);
  } else if (s.keys) {
    hipLaunchKernelGGL((attend_kernel<T, D, 2, true>), grid, dim3(64 * AT_WAVES), 0, st, a);
    hipLaunchKernelGGL((join_kernel<T, D, 32>), join, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((attend_kernel<T, D, 2, false>), grid, dim3(64 * AT_WAVES), 0, st, a);
    hipLaunchKernelGGL((join_kernel<T, D, 128>), join, dim3(256), 0, st, a);
  }
}

template <typename T>
static void launch_width(int64_t D, const Shape& s, const AttnArgs& a, hipStream_t st) {
  if (D == 64) launch<T, 64>(s, a, st);
  else if (D == 128) launch<T, 128>(s, a, st);
  else launch<T, 256>(s, a, st);
}

}  // namespace gdr

extern "C" {

int64_t macai_gdr_kv4_attention_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D) {
  if (T < 1 || B < 1 || Hk < 1 || Hq < Hk || D < 1) return 0;
  const gdr::Shape s = gdr::shape_for(T, B, Hq / Hk);
  const int64_t n = gdr::workers_for(s, D);
  return n * (int64_t)sizeof(int4) + 2 * n * s.rows() * (D + 4) * (int64_t)sizeof(float);
}

int macai_gdr_kv4_attention(const void* q, const uint8_t* cache, const int32_t* blocks, const int32_t* lens,
                            const int32_t* starts, void* o, void* workspace, int64_t T, int64_t B, int64_t W,
                            int64_t pages, int64_t page, int64_t Hq, int64_t Hk, int64_t D, int64_t q_row, int64_t q_head,
                            float scale, int32_t dtype, void* stream) {
  const char* what = "macai_gdr_kv4_attention";
  if (dtype < MACAI_GDR_F32 || dtype > MACAI_GDR_F16)
    return fail(MACAI_GDR_EUNSUP, "%s: dtype codes must be F32, BF16 or F16", what);
  if (D != 64 && D != 128 && D != 256)
    return fail(MACAI_GDR_EUNSUP, "%s: the head width must be 64, 128 or 256 (got %lld)", what, (long long)D);
  if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)
    return fail(MACAI_GDR_EUNSUP, "%s: a page must hold 16, 32, 64, 128 or 256 tokens (got %lld)", what, (long long)page);
  if (Hk < 1 || Hk > 1024 || Hq < Hk || Hq % Hk || Hq > 65536)
    return fail(MACAI_GDR_EINVAL, "%s: the key heads (%lld) must divide the query heads (%lld)", what, (long long)Hk,
                (long long)Hq);
  if (T < 1 || B < 1 || W < 1 || pages < 1 || T >= INT32_MAX / Hq || B >= INT32_MAX || pages >= INT64_C(1) << 31)
    return fail(MACAI_GDR_EINVAL, "%s: need T, B, W, pages >= 1 and T Hq, B, pages below 2^31", what);
  if (W > (INT32_MAX - 1024) / page) return fail(MACAI_GDR_EINVAL, "%s: a request's tokens must be below 2^31", what);
  if (!starts && T != B) return fail(MACAI_GDR_EINVAL, "%s: without starts every request has one query (T = B)", what);
  if (!q || !cache || !blocks || !lens || !o || !workspace) return fail(MACAI_GDR_EINVAL, "%s: null pointer", what);
  const void* ps[] = {q, cache, o, workspace};
  for (const void* p : ps)
    if (!aligned16(p)) return fail(MACAI_GDR_EINVAL, "%s: pointers must be 16-byte aligned", what);
  const int64_t v = dtype == MACAI_GDR_F32 ? 4 : 8;
  if (q_row % v || q_head % v) return fail(MACAI_GDR_EINVAL, "%s: strides must keep 16-byte alignment", what);
  const gdr::Shape s = gdr::shape_for(T, B, Hq / Hk);
  gdr::AttnArgs a{q, o, cache, blocks, lens, starts, nullptr, nullptr, q_row, q_head, T, B, W, pages, (int)Hq, (int)Hk,
                  (int)page, __builtin_ctzll((unsigned long long)page), gdr::workers_for(s, D), scale * 1.44269504088896341f};
  a.records = (int4*)workspace;
  a.part = (float*)((char*)workspace + a.workers * sizeof(int4));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MACAI_GDR_F32) gdr::launch_width<float>(D, s, a, st);
  else if (dtype == MACAI_GDR_BF16) gdr::launch_width<gdr::bf16>(D, s, a, st);
  else gdr::launch_width<gdr::f16>(D, s, a, st);
  return launched(what);
}

}  // extern "C"
