// Attention over packed rows for MI355X (gfx950), forward and backward, on the
// matrix cores: documents beside one another in a row, prefixes that see
// themselves both ways, scores capped by a tanh, a bias that falls with the
// distance. q, o, do [B, S, H, D], k, v [B, S, Hkv, D] bf16, heads of 64, 96 and
// 128, lse fp32 [B, H, S].
//
//   t_ij = cap tanh(scale q_i k_j / cap) - slope_h |i - j|      lo_i <= j < hi_i
//   p_ij = exp(t_ij - lse_i), o_i = sum_j p_ij v_j
//   dt_ij = p_ij (do_i v_j - do_i o_i), ds_ij = dt_ij (1 - tanh^2)
//
// Every mask is an interval of keys for a query, lo and hi growing with the query,
// and with that an interval of queries for a key (spans_kernel): a tile of either
// is skipped, taken whole or compared element by element by the ends of its first
// and last rows alone, and what is skipped costs nothing. Layout of the products,
// order of the contracted index and the two passes of the backward are those of
// attention.hip, which says why.
//
// The matrix cores add 0 times what a hidden row holds, which is no 0 for an
// infinity or NaN there: a row whose sums are not finite though all that it sees is,
// by its statistics or by a look, is summed again over that alone (the loops over
// `bad` below, which nothing reaches with finite inputs, and of the rest only rows that
// share a tile with something hidden that is not finite).

#include "attention_tile.h"
#include "ds_kernels.h"

namespace {

using namespace attn;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -__FLT_MAX__;     // a maximum before anything was seen
typedef int i32x2 __attribute__((ext_vector_type(2)));

struct View {             // element strides of [B, S, H, D]
  long long b, s, h;
};

struct Args {
  const short *q, *k, *v, *o, *dout;
  short *out, *dq, *dk, *dv;
  float* lse;             // in units of log2
  int* rest;              // [B, S, H, D] bytes: what `out` was rounded by, or null
  float* stat;            // [B, H, S]: sum(do * o), from dQ's pass to dK's
  float* part;            // splits of dK and dV, or null
  const int* spans;       // [4][B, S]: q lo, q hi, k lo, k hi, or null
  const float* slopes;    // [H]
  View vq, vk, vv, vo, vd;
  int B, S, H, Hkv, causal;
  float scale, c;         // c: scale * log2(e)
  float a, cap;           // a: 2 log2(e) scale / cap, cap: cap * log2(e)
  float x;                // scale / cap
};

struct Span {
  int lo, hi;
};

// Keys that query i sees, or queries that see key i: inside the row whatever the spans
// hold, both ends, since a difference of ends anywhere may wrap to a positive one.
__device__ __forceinline__ Span span(const Args& a, int b, int i, bool key) {
  Span s;
  if (a.spans != nullptr) {
    const long long n = (long long)a.B * a.S;
    const int* p = a.spans + (key ? 2 * n : 0) + (long long)b * a.S + i;
    s.lo = min(max(p[0], 0), a.S);
    s.hi = min(max(p[n], 0), a.S);
  } else {
    s.lo = key && a.causal ? i : 0;
    s.hi = !key && a.causal ? i + 1 : a.S;
  }
  return s;
}

__device__ __forceinline__ int uni(int x) {
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int lane_of(int x, int lane) {
  return __builtin_amdgcn_readlane(x, lane);
}
__device__ __forceinline__ float value(short x) {
  return __builtin_bit_cast(float, (unsigned)(unsigned short)x << 16);
}
__device__ __forceinline__ bool finite(float x) {
  return __builtin_fabsf(x) < __builtin_inff();
}

// t and the eight numbers of an operand.
__device__ __forceinline__ float add_pairs(s16x8 x, float t) {
  const b16x8 y = __builtin_bit_cast(b16x8, x);
  const b16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t = __builtin_amdgcn_fdot2_f32_bf16(b16x2{y[2 * i], y[2 * i + 1]}, one, t,
                                        false);
  return t;
}

// Scores in units of log2, with their derivative's factor where that is asked for.
// tanh x = 1 - 2 / (e^2x + 1) holds for every x, infinities among them. (A polynomial
// where all of a tile's scores are near 0 takes two thirds of its instructions and was
// 4% less of the forward and nothing of the rest: the matrix cores' operands, not
// these, are what a step waits for.)
// That 1 - 2 / (..) is off by 2^-23 of the cap, wherever x is: nothing beside bf16 for
// caps up to 200. WIDE ones take the series of tanh up to x of 1/4, to 3e-7 of itself.
enum Cap { NONE, USUAL, WIDE };

template <int CAP, bool BIAS>
struct Score {
  const Args& a;
  const float slope;
  __device__ __forceinline__ float operator()(float s, float far,
                                              float& bend) const {
    float t;
    if (CAP) {
      const float r =
          __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * a.a) + 1.f);
      t = __builtin_fmaf(-2.f * a.cap, r, a.cap);
      bend = 4.f * r * (1.f - r);
      if (CAP == WIDE) {
        const float x = s * a.x, y = x * x;
        float p = __builtin_fmaf(y, -17.f / 315, 2.f / 15);
        p = __builtin_fmaf(y, p, -1.f / 3);
        p = __builtin_fmaf(y, p, 1.f);
        if (__builtin_fabsf(x) < 0.25f) t = s * a.c * p;
      }
    } else {
      t = s * a.c;
    }
    if (BIAS) t = __builtin_fmaf(-__builtin_fabsf(far), slope, t);
    return t;
  }
};

// Workgroup -> (block of rows, batch * head): each XCD takes an eighth of the
// heads, whose keys and values its L2 then holds.
__device__ __forceinline__ void place(int id, int blocks, int heads, int& blk,
                                      int& bh) {
  if (heads % 8 == 0) {
    const int per = heads / 8, k = id >> 3;
    blk = k / per;
    bh = (id & 7) * per + k % per;
  } else {
    blk = id / heads;
    bh = id % heads;
  }
}

// The sum of two rows' products, each lane its coordinates lane and lane + 64.
template <int D>
__device__ __forceinline__ float dot(const short* x, const short* y, int lane) {
  float t = lane < D ? value(x[lane]) * value(y[lane]) : 0.f;
  if (lane + 64 < D) t += value(x[lane + 64]) * value(y[lane + 64]);
  return ds::wave_reduce_sum(t);
}

// sum(do * o) of the backward is taken from gradients it is nearly as large as, where
// scores are far apart: from an o rounded to bf16 it is what dQ and dK are most off by
// (0.0023 of them of 0.0033 in all, scores of a deviation of 4). So the forward keeps
// the next eight bits of o as well, a signed byte each: bits of an fp32 o = those of
// its bf16 + 256 times the byte.
__device__ __forceinline__ unsigned rest_of(float x, int high) {
  const int d = (__builtin_bit_cast(int, x) - high + 128) >> 8;
  return (unsigned)min(max(d, -128), 127) & 255u;
}
__device__ __forceinline__ unsigned rests(float a, float b, int ab, float c,
                                          float d, int cd) {
  return rest_of(a, ab << 16) | rest_of(b, ab & 0xffff0000) << 8 |
         rest_of(c, cd << 16) << 16 | rest_of(d, cd & 0xffff0000) << 24;
}

// What rounding to the operand x left of it, as another. The scores' gradients take both:
// those of a row add up to 0, so that dQ and dK are small beside the sums of what they
// are made of, and with a rounding of 2^-8 they were off 64 bits by 1.41 of their own
// rounding's 0.00166 where scores lie close together and up to 1.56 where they lie a
// deviation of 4 apart, capped or not; with both by 1.02 to 1.12. That is 4 to 9% of a
// training step's time. The weights are positive and add up to 1: o and dV are off by
// 1.0 to 1.28 and by 1.28 to 1.42, and both for them too would be another 8 to 15%.
__device__ __forceinline__ s16x8 rounded_off(const f32x16& p, int s, s16x8 x) {
  f32x16 left;
#pragma unroll
  for (int r = 0; r < 8; ++r) left[8 * s + r] = p[8 * s + r] - value(x[r]);
  return operand(left, s);
}

// Loads into registers end here, before a loop: the compiler, which does not know of the
// tiles' loads, would wait for these where it first uses them, in every step of the
// loop, and so for the next tile's as well.
template <int N>
__device__ __forceinline__ void settle(s16x8 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// ------------------------------------------------------------------ forward
//
// 4 waves of 32 query rows walk the keys that any of them sees, 32 or 64 a step, K and V
// double-buffered in LDS by direct loads. Three workgroups a CU (two of heads of 64's
// four), so that one's first loads and last stores lie behind another's products: a
// document of a few hundred tokens is seven steps of a workgroup. Bound by the vector
// unit (74% busy, and the matrix cores 36%, at the 2.0 GHz that the power leaves). us:
// 1 x 8192 capped, 32 on 8 heads of 128 732 (751 TFLOP/s); nine documents in 4 x 4096 225
// (385 of what is seen, 1.19 times that computed); 8 x 1999, eleven documents of 12
// heads of 64 with the bias 56; 2 x 4096 capped, four with prefixes, 32 heads of 96 246.
// The first kernel, eight waves and steps of 64, took 862, 263, 56 and 273.

template <int D, int CAP, bool BIAS, int NW, int KB>
__global__ __launch_bounds__(NW * 64, KB == 32 ? 3 : 2) void fwd_kernel(
    const Args a, const int blocks, const int heads) {
  constexpr int KT = KB / 32, DB = D / 32, KK = D / 16;
  constexpr int QB = 32 * NW, TPB = 64 * NW;
  constexpr bool PLAIN = !CAP && !BIAS;
  using T = Tile<D, true>;
  __shared__ __attribute__((aligned(16))) short kt[2][KB * T::SC * 8];
  __shared__ __attribute__((aligned(16))) short vt[2][KB * T::SC * 8];

  const int tid = threadIdx.x, lane = tid & 63, wid = uni(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int ra = T::rows_at(lane), ca = T::cols_at(lane);
  const int S = a.S;
  int blk, bh;
  place(blockIdx.x, blocks, heads, blk, bh);
  blk = blocks - 1 - blk;
  const int b = bh / a.H, h = bh % a.H, hkv = h / (a.H / a.Hkv);
  const int q0b = blk * QB, q0 = q0b + wid * 32, row = q0 + col;
  const int at = min(row, S - 1);

  const short* kp = a.k + b * a.vk.b + hkv * a.vk.h;
  const short* vp = a.v + b * a.vv.b + hkv * a.vv.h;
  const short* qp = a.q + b * a.vq.b + h * a.vq.h + at * a.vq.s;
  const Score<CAP, BIAS> score = {a, BIAS ? a.slopes[h] * LOG2E : 0.f};
  const float c = PLAIN ? a.c : 1.f;
  const Span me = span(a, b, at, false);
  const int width = max(me.hi - me.lo, 0);
  // of the wave: what anyone sees, and what everyone does
  const int any0 = lane_of(me.lo, 0), all0 = lane_of(me.lo, 31);
  const int all1 = lane_of(me.hi, 0);
  const int any1 = q0 < S ? lane_of(me.hi, 31) : 0;
  const int k_begin = uni(span(a, b, q0b, false).lo);
  const int k_end = uni(span(a, b, min(q0b + QB - 1, S - 1), false).hi);
  const int steps = (k_end - k_begin + KB - 1) / KB;

  // sums of the weights, and of the weights as they are rounded for the product: o is
  // over these, so that the rounding of a weight that is most of its row goes out
  float m = LOWEST, l = 0.f, lr = 0.f;
  f32x16 acc[DB] = {};
  auto fetch = [&](int k0, int buf) __attribute__((always_inline)) {
    T::template fetch<KB, TPB>(kp + k0 * a.vk.s, (int)a.vk.s, S - k0, kt[buf],
                               tid);
    T::template fetch<KB, TPB>(vp + k0 * a.vv.s, (int)a.vv.s, S - k0, vt[buf],
                               tid);
  };
  // the queries behind the first tile: one wait for both
  if (steps > 0) fetch(k_begin, 0);
  s16x8 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = *(const s16x8*)(qp + 16 * kk + 8 * half);
  arrive();
  settle(qf);
  for (int it = 0; it < steps; ++it) {
    const int k0 = k_begin + it * KB, cur = it & 1;
    if (it + 1 < steps) fetch(k0 + KB, cur ^ 1);
    if (k0 < any1 && k0 + KB > any0) {
      f32x16 p[KT] = {};
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          p[t] = mfma(T::rows(kt[cur], 32 * t, kk, ra), qf[kk], p[t]);
      __builtin_amdgcn_s_setprio(0);
      if (!PLAIN) {
        const float far = (float)(k0 + 4 * half - at);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float bend;
            p[t][r] = score(
                p[t][r], far + (32 * t + (r & 3) + 8 * (r >> 2)), bend);
          }
      }
      if (k0 < all0 || k0 + KB > all1) {
        const int first = me.lo - k0 - 4 * half;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((unsigned)(32 * t + (r & 3) + 8 * (r >> 2) - first) >=
                (unsigned)width)
              p[t][r] = -__builtin_inff();
      }
      float mt = LOWEST;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, p[t][r]);
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      if (!__all((mt - m) * c <= 8.f)) {
        const float mn = fmaxf(m, mt);
        const float alpha = __builtin_amdgcn_exp2f((m - mn) * c);
        m = mn;
        l *= alpha;
        lr *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
      }
      // before anything was seen not infinite, which hidden scores of -inf would meet
      const float mc = PLAIN ? fmaxf(m * c, LOWEST) : m;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float x0 = PLAIN ? __builtin_fmaf(p[t][r], c, -mc)
                                 : p[t][r] - m;
          const float x1 = PLAIN ? __builtin_fmaf(p[t][r + 1], c, -mc)
                                 : p[t][r + 1] - m;
          p[t][r] = __builtin_amdgcn_exp2f(x0);
          p[t][r + 1] = __builtin_amdgcn_exp2f(x1);
          l0 += p[t][r];
          l1 += p[t][r + 1];
        }
      l += l0 + l1;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const s16x8 pb = operand(p[t], s);
          lr = add_pairs(pb, lr);
#pragma unroll
          for (int db = 0; db < DB; ++db)
            acc[db] =
                mfma(T::cols(vt[cur], 32 * t + 16 * s, db, ca), pb, acc[db]);
        }
      __builtin_amdgcn_s_setprio(0);
    }
    arrive();
  }

  l += __shfl_xor(l, 32, 64);
  lr += __shfl_xor(lr, 32, 64);
  // a row that sees nothing is 0, and its logarithm of nothing -inf
  const float inv = width == 0 ? 0.f : 1.f / lr;
  bool good = true;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      acc[db][r] = width == 0 ? 0.f : acc[db][r] * inv;
      good = good && finite(acc[db][r]);
    }
  const bool real = row < S;
  const float sum = m * c + __builtin_amdgcn_logf(l);      // log2
  if (real && half == 0)
    a.lse[((long long)b * a.H + h) * S + row] =
        width == 0 ? -__builtin_inff() : sum;
  short* const op = a.out + b * a.vo.b + h * a.vo.h;
  if (real) {
    short* y = op + row * a.vo.s + 4 * half;
    int* z = a.rest +
             ((((long long)b * S + row) * a.H + h) * D + 4 * half) / 4;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float *x = (const float*)&acc[db] + 4 * g;
        const i32x2 w = {pack2(x[0], x[1]), pack2(x[2], x[3])};
        *(i32x2*)(y + 32 * db + 8 * g) = w;
        if (a.rest != nullptr)
          z[8 * db + 2 * g] =
              (int)rests(x[0], x[1], w[0], x[2], x[3], w[1]);
      }
  }
  unsigned long long bad = __ballot(real && !good && finite(sum));
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) {
    // the first and the last of the wave's keys whose value is not finite: a row that
    // sees one of them is as it is
    int low = S, high = -1;
    for (int j = any0 + lane; j < any1; j += 64) {
      const short* vj = vp + j * a.vv.s;
      bool sick = false;
      for (int d = 0; d < D; ++d) sick = sick || !finite(value(vj[d]));
      if (sick) {
        low = min(low, j);
        high = j;
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      low = min(low, __shfl_xor(low, off, 64));
      high = max(high, __shfl_xor(high, off, 64));
    }
    const bool sees = (low >= me.lo && low < me.hi) ||
                      (high >= me.lo && high < me.hi);
    bad &= ~__ballot(sees);
    __builtin_amdgcn_s_waitcnt(0);      // the rows as they were written
  }
  for (; bad; bad &= bad - 1) {
    const int n = __builtin_ctzll(bad), i = q0 + n;
    const int lo = lane_of(me.lo, n), hi = lane_of(me.hi, n);
    const float z = __builtin_bit_cast(
        float, lane_of(__builtin_bit_cast(int, sum), n));
    const short* qi = a.q + b * a.vq.b + h * a.vq.h + i * a.vq.s;
    float y0 = 0.f, y1 = 0.f;
    for (int j = lo; j < hi; ++j) {
      float bend;
      const float t = score(dot<D>(kp + j * a.vk.s, qi, lane), (float)(j - i),
                            bend);
      const float p = __builtin_amdgcn_exp2f(t - z);
      const short* vj = vp + j * a.vv.s;
      if (lane < D) y0 += p * value(vj[lane]);
      if (lane + 64 < D) y1 += p * value(vj[lane + 64]);
    }
    short* y = op + i * a.vo.s;
    char* r = (char*)a.rest + (((long long)b * S + i) * a.H + h) * D;
    const int w = pack2(y0, y1);
    if (lane < D) y[lane] = (short)w;
    if (lane + 64 < D) y[lane + 64] = (short)(w >> 16);
    if (a.rest != nullptr) {
      if (lane < D) r[lane] = (char)rest_of(y0, w << 16);
      if (lane + 64 < D) r[lane + 64] = (char)rest_of(y1, w & 0xffff0000);
    }
  }
}

// ----------------------------------------------------------------- backward

// Both passes compute S and dP again, as attention.hip's: every sum in registers and in
// one order, no atomics. dQ goes first and leaves sum(do * o) for the other: a kernel for
// these alone read do once more (54 us of the nine documents' 930 in all). Bound by the
// matrix and vector units together for one long document (42 to 46 and 57 to 66% busy),
// by waves that wait for the rest of their workgroup for many (27 to 30 and 27%); waves of
// two or eight to a tile, a half's products beside the other half's arithmetic or
// prefetched operands are all slower. us, cases as above: dQ 1182 (930 TFLOP/s of its
// products, four with what a rounding leaves), 345, 74, 377; dK and dV 1575 and 47 for the
// splits' sums (873 of five), 387, 86, 414.
//
// dK and dV: a wave owns 32 keys and walks the queries that see them.
template <int D, int CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void dkdv_kernel(const Args a,
                                                      const int blocks,
                                                      const int heads) {
  constexpr int QB = 64, DB = D / 32, KK = D / 16;
  constexpr bool PLAIN = !CAP && !BIAS;
  using T = Tile<D, true>;
  __shared__ __attribute__((aligned(16))) short qt[2][QB * T::SC * 8];
  __shared__ __attribute__((aligned(16))) short dt[2][QB * T::SC * 8];
  __shared__ __attribute__((aligned(16))) float st[2][2][QB];

  const int tid = threadIdx.x, lane = tid & 63, wid = uni(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int ra0 = T::rows_at(lane), ca0 = T::cols_at(lane);
  const int S = a.S;
  int blk, bh;
  place(blockIdx.x, blocks, heads, blk, bh);
  const int b = bh / a.Hkv, hkv = bh % a.Hkv, G = a.H / a.Hkv;
  const int k0b = blk * 128, k0 = k0b + wid * 32, key = k0 + col;
  const int at = min(key, S - 1);

  f32x16 dka[DB] = {}, dva[DB] = {};

  const Span me = span(a, b, at, true);
  const int width = max(me.hi - me.lo, 0);
  const int any0 = lane_of(me.lo, 0), all0 = lane_of(me.lo, 31);
  const int all1 = lane_of(me.hi, 0);
  const int any1 = k0 < S ? lane_of(me.hi, 31) : 0;
  const int first = uni(span(a, b, k0b, true).lo);
  const int last = uni(span(a, b, min(k0b + 127, S - 1), true).hi);
  const int per = max((last - first + QB - 1) / QB, 0);
  const int g0 = blockIdx.y * G / gridDim.y;
  const int g1 = (blockIdx.y + 1) * G / gridDim.y;
  const int steps = (g1 - g0) * per;

  auto fetch = [&](int h, int s0, int buf, int tid)
                   __attribute__((always_inline)) {
    T::template fetch<QB, 256>(a.q + b * a.vq.b + h * a.vq.h + s0 * a.vq.s,
                               (int)a.vq.s, S - s0, qt[buf], tid);
    T::template fetch<QB, 256>(a.dout + b * a.vd.b + h * a.vd.h + s0 * a.vd.s,
                               (int)a.vd.s, S - s0, dt[buf], tid);
    if (wid < 2) {
      const float* p = (wid ? a.stat : a.lse) +
                       ((long long)b * a.H + h) * S + s0;
      load_lds<4>(p, 4u * min(lane, S - s0 - 1), lds_at(&st[buf][wid][0]));
    }
  };

  int h = hkv * G + g0, s0 = first;
  if (steps > 0) fetch(h, s0, 0, tid);
  const short* kp = a.k + b * a.vk.b + hkv * a.vk.h + at * a.vk.s;
  const short* vp = a.v + b * a.vv.b + hkv * a.vv.h + at * a.vv.s;
  s16x8 kf[KK], vf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    kf[kk] = *(const s16x8*)(kp + 16 * kk + 8 * half);
    vf[kk] = *(const s16x8*)(vp + 16 * kk + 8 * half);
  }
  arrive();
  settle(kf);
  settle(vf);
  for (int it = 0; it < steps; ++it) {
    const int cur = it & 1;
    const Score<CAP, BIAS> score = {a, BIAS ? a.slopes[h] * LOG2E : 0.f};
    int s1 = s0 + QB;
    if (s1 >= last) {
      s1 = first;
      ++h;
    }
    if (it + 1 < steps) {
      int tid_ = tid;
      asm("" : "+v"(tid_));
      fetch(h, s1, cur ^ 1, tid_);
    }
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const int r0 = s0 + 32 * t;
      if (r0 >= any1 || r0 + 32 <= any0) continue;
      int ra = ra0, ca = ca0;      // kept out of registers that the loop needs
      asm("" : "+v"(ra), "+v"(ca));
      f32x16 p = {}, dp = {};
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        p = mfma(T::rows(qt[cur], 32 * t, kk, ra), kf[kk], p);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        dp = mfma(T::rows(dt[cur], 32 * t, kk, ra), vf[kk], dp);
      __builtin_amdgcn_s_setprio(0);
      const float far = (float)(r0 + 4 * half - at);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = 32 * t + 8 * g + 4 * half;
        const f32x4 ls = *(const f32x4*)&st[cur][0][i];
        const f32x4 dl = *(const f32x4*)&st[cur][1][i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          float bend = 1.f;
          const float x = PLAIN
                              ? __builtin_fmaf(p[r], a.c, -ls[e])
                              : score(
                                    p[r], far + (8 * g + e), bend) - ls[e];
          p[r] = __builtin_amdgcn_exp2f(x);
          dp[r] -= dl[e];
          if (CAP) dp[r] *= bend;
          dp[r] *= p[r];
        }
      }
      if (r0 < all0 || r0 + 32 > all1) {
        const int from = me.lo - r0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((unsigned)((r & 3) + 8 * (r >> 2) - from) >= (unsigned)width) {
            p[r] = 0.f;
            dp[r] = 0.f;
          }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s16x8 pb = operand(p, s);
#pragma unroll
        for (int db = 0; db < DB; ++db)
          dva[db] =
              mfma(T::cols(dt[cur], 32 * t + 16 * s, db, ca), pb, dva[db]);
        const s16x8 sb = operand(dp, s), lb = rounded_off(dp, s, sb);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const s16x8 qc = T::cols(qt[cur], 32 * t + 16 * s, db, ca);
          dka[db] = mfma(qc, sb, dka[db]);
          dka[db] = mfma(qc, lb, dka[db]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    arrive();
    s0 = s1;
  }

  bool good = true;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      good = good && finite(dka[db][r]) && finite(dva[db][r]);
  const bool real = key < S;
  const long long n = (long long)a.B * S * a.Hkv * D;
  const long long row_at = ((long long)b * S * a.Hkv + hkv) * D;
  const long long step = (long long)a.Hkv * D;
  float* const part = a.part ? a.part + 2 * n * blockIdx.y + row_at : nullptr;
  if (real && part != nullptr) {       // added up by add_kernel
    float* pp = part + key * step + 4 * half;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        *(f32x4*)(pp + 32 * db + 8 * g) =
            f32x4{dka[db][4 * g], dka[db][4 * g + 1], dka[db][4 * g + 2],
                  dka[db][4 * g + 3]};
        *(f32x4*)(pp + n + 32 * db + 8 * g) =
            f32x4{dva[db][4 * g], dva[db][4 * g + 1], dva[db][4 * g + 2],
                  dva[db][4 * g + 3]};
      }
  } else if (real) {
    short* dkp = a.dk + row_at + key * step + 4 * half;
    short* dvp = a.dv + row_at + key * step + 4 * half;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        *(i32x2*)(dkp + 32 * db + 8 * g) =
            i32x2{pack2(dka[db][4 * g] * a.scale, dka[db][4 * g + 1] * a.scale),
                  pack2(dka[db][4 * g + 2] * a.scale,
                        dka[db][4 * g + 3] * a.scale)};
        *(i32x2*)(dvp + 32 * db + 8 * g) =
            i32x2{pack2(dva[db][4 * g], dva[db][4 * g + 1]),
                  pack2(dva[db][4 * g + 2], dva[db][4 * g + 3])};
      }
  }
  unsigned long long bad = __ballot(real && !good);
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) __builtin_amdgcn_s_waitcnt(0);
  for (; bad; bad &= bad - 1) {
    const int w = __builtin_ctzll(bad), j = k0 + w;
    const int lo = lane_of(me.lo, w), hi = lane_of(me.hi, w);
    bool sick = false;      // a row that sees the key
    for (int head = hkv * G + g0; head < hkv * G + g1; ++head)
      for (int i = lo + lane; i < hi; i += 64) {
        const long long u = ((long long)b * a.H + head) * S + i;
        sick = sick || !finite(a.lse[u]) || !finite(a.stat[u]);
      }
    if (__any(sick)) continue;
    const short* kj = a.k + b * a.vk.b + hkv * a.vk.h + j * a.vk.s;
    const short* vj = a.v + b * a.vv.b + hkv * a.vv.h + j * a.vv.s;
    float k_0 = 0.f, k_1 = 0.f, v_0 = 0.f, v_1 = 0.f;
    for (int head = hkv * G + g0; head < hkv * G + g1; ++head) {
      const Score<CAP, BIAS> score = {a, BIAS ? a.slopes[head] * LOG2E : 0.f};
      const float* ls = a.lse + ((long long)b * a.H + head) * S;
      const float* dl = a.stat + ((long long)b * a.H + head) * S;
      for (int i = lo; i < hi; ++i) {
        const short* qi = a.q + b * a.vq.b + head * a.vq.h + i * a.vq.s;
        const short* di = a.dout + b * a.vd.b + head * a.vd.h + i * a.vd.s;
        float bend = 1.f;
        const float t = score(dot<D>(qi, kj, lane), (float)(i - j), bend);
        const float p = __builtin_amdgcn_exp2f(t - ls[i]);
        float ds = (dot<D>(di, vj, lane) - dl[i]) * p;
        if (CAP) ds *= bend;
        if (lane < D) {
          k_0 += ds * value(qi[lane]);
          v_0 += p * value(di[lane]);
        }
        if (lane + 64 < D) {
          k_1 += ds * value(qi[lane + 64]);
          v_1 += p * value(di[lane + 64]);
        }
      }
    }
    if (part != nullptr) {
      float* pp = part + j * step;
      if (lane < D) {
        pp[lane] = k_0;
        pp[n + lane] = v_0;
      }
      if (lane + 64 < D) {
        pp[lane + 64] = k_1;
        pp[n + lane + 64] = v_1;
      }
    } else {
      short* dkp = a.dk + row_at + j * step;
      short* dvp = a.dv + row_at + j * step;
      if (lane < D) {
        dkp[lane] = (short)pack2(k_0 * a.scale, 0.f);
        dvp[lane] = (short)pack2(v_0, 0.f);
      }
      if (lane + 64 < D) {
        dkp[lane + 64] = (short)pack2(k_1 * a.scale, 0.f);
        dvp[lane + 64] = (short)pack2(v_1, 0.f);
      }
    }
  }
}

// dK and dV from the partial sums of the splits: part [splits][dk, dv][n].
__global__ __launch_bounds__(256) void add_kernel(
    const float* __restrict__ part, short* __restrict__ dk,
    short* __restrict__ dv, const long long n, const int splits,
    const float scale) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= 2 * n) return;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) t += *(const f32x4*)(part + 2 * n * s + i);
  const bool is_k = i < n;
  if (is_k) t *= scale;
  *(i32x2*)((is_k ? dk + i : dv + (i - n))) =
      i32x2{pack2(t[0], t[1]), pack2(t[2], t[3])};
}

// dQ: a wave owns 32 queries and walks the keys that they see.
template <int D, int CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void dq_kernel(const Args a,
                                                    const int blocks,
                                                    const int heads) {
  constexpr int KB = 64, DB = D / 32, KK = D / 16;
  constexpr bool PLAIN = !CAP && !BIAS;
  using T = Tile<D, true>;
  __shared__ __attribute__((aligned(16))) short kt[2][KB * T::SC * 8];
  __shared__ __attribute__((aligned(16))) short vt[2][KB * T::SC * 8];

  const int tid = threadIdx.x, lane = tid & 63, wid = uni(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int ra = T::rows_at(lane), ca = T::cols_at(lane);
  const int S = a.S;
  int blk, bh;
  place(blockIdx.x, blocks, heads, blk, bh);
  blk = blocks - 1 - blk;
  const int b = bh / a.H, h = bh % a.H, hkv = h / (a.H / a.Hkv);
  const int q0b = blk * 128, q0 = q0b + wid * 32, row = q0 + col;
  const int at = min(row, S - 1);
  const short* kp = a.k + b * a.vk.b + hkv * a.vk.h;
  const short* vp = a.v + b * a.vv.b + hkv * a.vv.h;
  const short* qb = a.q + b * a.vq.b + h * a.vq.h;
  const short* db_ = a.dout + b * a.vd.b + h * a.vd.h;

  f32x16 acc[DB] = {};

  const Score<CAP, BIAS> score = {a, BIAS ? a.slopes[h] * LOG2E : 0.f};
  const Span me = span(a, b, at, false);
  const int width = max(me.hi - me.lo, 0);
  const int any0 = lane_of(me.lo, 0), all0 = lane_of(me.lo, 31);
  const int all1 = lane_of(me.hi, 0);
  const int any1 = q0 < S ? lane_of(me.hi, 31) : 0;
  const int k_begin = uni(span(a, b, q0b, false).lo);
  const int k_end = uni(span(a, b, min(q0b + 127, S - 1), false).hi);
  const int steps = (k_end - k_begin + KB - 1) / KB;

  auto fetch = [&](int k0, int buf) __attribute__((always_inline)) {
    T::template fetch<KB, 256>(kp + k0 * a.vk.s, (int)a.vk.s, S - k0, kt[buf],
                               tid);
    T::template fetch<KB, 256>(vp + k0 * a.vv.s, (int)a.vv.s, S - k0, vt[buf],
                               tid);
  };
  // the rows behind the first tile: one wait for all
  if (steps > 0) fetch(k_begin, 0);
  s16x8 qf[KK], df[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    qf[kk] = *(const s16x8*)(qb + at * a.vq.s + 16 * kk + 8 * half);
    df[kk] = *(const s16x8*)(db_ + at * a.vd.s + 16 * kk + 8 * half);
  }
  const long long sat = ((long long)b * a.H + h) * S + at;
  const float ls = a.lse[sat];
  float dl = 0.f;
  {
    const short* op = a.o + b * a.vo.b + h * a.vo.h + at * a.vo.s;
    const int* rp = a.rest + (((long long)b * S + at) * a.H + h) * (D / 4);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const s16x8 y = *(const s16x8*)(op + 16 * kk + 8 * half);
      const i32x2 r = *(const i32x2*)(rp + 4 * kk + 2 * half);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int more = (r[e >> 2] << (24 - 8 * (e & 3))) >> 24;   // signed
        const int o = ((int)(unsigned short)y[e] << 16) + more * 256;
        dl = __builtin_fmaf(value(df[kk][e]), __builtin_bit_cast(float, o), dl);
      }
    }
    dl += __shfl_xor(dl, 32, 64);
    if (row < S && half == 0) a.stat[sat] = dl;
  }
  arrive();
  settle(qf);
  settle(df);
  for (int it = 0; it < steps; ++it) {
    const int k0 = k_begin + it * KB, cur = it & 1;
    if (it + 1 < steps) fetch(k0 + KB, cur ^ 1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key0 = k0 + 32 * t;
      if (key0 >= any1 || key0 + 32 <= any0) continue;
      f32x16 p = {}, dp = {};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        p = mfma(T::rows(kt[cur], 32 * t, kk, ra), qf[kk], p);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        dp = mfma(T::rows(vt[cur], 32 * t, kk, ra), df[kk], dp);
      const float far = (float)(key0 + 4 * half - at);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float bend = 1.f;
        const float x =
            PLAIN ? __builtin_fmaf(p[r], a.c, -ls)
                  : score(
                        p[r], far + ((r & 3) + 8 * (r >> 2)), bend) - ls;
        dp[r] -= dl;
        if (CAP) dp[r] *= bend;
        dp[r] *= __builtin_amdgcn_exp2f(x);
      }
      if (key0 < all0 || key0 + 32 > all1) {
        const int first = me.lo - key0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((unsigned)((r & 3) + 8 * (r >> 2) - first) >= (unsigned)width)
            dp[r] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s16x8 sb = operand(dp, s);
        const s16x8 lb = rounded_off(dp, s, sb);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const s16x8 kc = T::cols(kt[cur], 32 * t + 16 * s, db, ca);
          acc[db] = mfma(kc, sb, acc[db]);
          acc[db] = mfma(kc, lb, acc[db]);
        }
      }
    }
    arrive();
  }

  bool good = true;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) good = good && finite(acc[db][r]);
  const bool real = row < S;
  const long long step = (long long)a.H * D;
  short* const dqp = a.dq + ((long long)b * S * a.H + h) * D;
  if (real) {
    short* y = dqp + row * step + 4 * half;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(i32x2*)(y + 32 * db + 8 * g) =
            i32x2{pack2(acc[db][4 * g] * a.scale, acc[db][4 * g + 1] * a.scale),
                  pack2(acc[db][4 * g + 2] * a.scale,
                        acc[db][4 * g + 3] * a.scale)};
  }
  unsigned long long bad =
      __ballot(real && !good && (width == 0 || (finite(ls) && finite(dl))));
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) __builtin_amdgcn_s_waitcnt(0);
  for (; bad; bad &= bad - 1) {
    const int n = __builtin_ctzll(bad), i = q0 + n;
    const int lo = lane_of(me.lo, n), hi = lane_of(me.hi, n);
    const float z = __builtin_bit_cast(
        float, lane_of(__builtin_bit_cast(int, ls), n));
    const float own = __builtin_bit_cast(
        float, lane_of(__builtin_bit_cast(int, dl), n));
    const short *qi = qb + i * a.vq.s, *di = db_ + i * a.vd.s;
    float y0 = 0.f, y1 = 0.f;
    for (int j = lo; j < hi; ++j) {
      const short* kj = kp + j * a.vk.s;
      float bend = 1.f;
      const float t = score(dot<D>(kj, qi, lane), (float)(j - i), bend);
      float ds = (dot<D>(vp + j * a.vv.s, di, lane) - own) *
                 __builtin_amdgcn_exp2f(t - z);
      if (CAP) ds *= bend;
      if (lane < D) y0 += ds * value(kj[lane]);
      if (lane + 64 < D) y1 += ds * value(kj[lane + 64]);
    }
    short* y = dqp + i * step;
    if (lane < D) y[lane] = (short)pack2(y0 * a.scale, 0.f);
    if (lane + 64 < D) y[lane + 64] = (short)pack2(y1 * a.scale, 0.f);
  }
}

// ------------------------------------------------------------------- spans
//
// Of a document of the rows s .. e - 1 with a prefix of p: a query i sees the keys
// s .. max(i + 1, s + p) - 1 (causal) or s .. e - 1, a key j is seen by the queries
// from j on, or of the prefix from s on. Rows of no document see nothing and stand
// at themselves, which keeps all four growing. A thread a row; the document's ends
// past the workgroup's own rows are looked for 4096 rows at a time. 3 to 7 us (4 x 4096,
// 1 x 8192), once a batch.

constexpr int ST = 1024, FAR = 4 * ST;

template <typename I>
__global__ __launch_bounds__(ST) void spans_kernel(
    const I* __restrict__ ids, const int* __restrict__ prefix,
    int* __restrict__ spans, const int B, const int S, const int N,
    const int causal) {
  __shared__ int first[ST / 64], last[ST / 64], out[2];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int b = blockIdx.y, r0 = blockIdx.x * ST, i = r0 + tid;
  const I* row = ids + (long long)b * S;
  auto begins = [&](int j) { return j == 0 || row[j] != row[j - 1]; };

  const bool here = i < S && begins(i);
  // the last beginning up to a lane, the first behind it
  const unsigned long long mask = __ballot(here);
  const unsigned long long upto = mask & (~0ull >> (63 - lane));
  const unsigned long long behind = lane == 63 ? 0 : mask >> (lane + 1);
  if (lane == 0) {
    last[wid] = mask ? r0 + wid * 64 + 63 - __builtin_clzll(mask) : -1;
    first[wid] = mask ? r0 + wid * 64 + __builtin_ctzll(mask) : S;
  }
  if (tid < 2) out[tid] = tid == 0 ? -1 : S;
  __syncthreads();
  // where the document that reaches into these rows began
  for (int hi = r0; hi > 0;) {
    const int lo = max(hi - FAR, 0);
    int found = -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = lo + u * ST + tid;
      if (j < hi && begins(j)) found = j;
    }
    if (found >= 0) atomicMax(&out[0], found);
    __syncthreads();
    if (out[0] >= 0) break;
    hi = lo;
    __syncthreads();
  }
  // and where the one that goes on behind them ends
  for (int lo = r0 + ST; lo < S; lo += FAR) {
    int found = S;
#pragma unroll
    for (int u = 3; u >= 0; --u) {
      const int j = lo + u * ST + tid;
      if (j < S && begins(j)) found = j;
    }
    if (found < S) atomicMin(&out[1], found);
    __syncthreads();
    if (out[1] < S) break;
    __syncthreads();
  }
  if (i >= S) return;
  int s = upto ? r0 + wid * 64 + 63 - __builtin_clzll(upto) : -1;
  for (int w = wid - 1; s < 0 && w >= 0; --w) s = last[w];
  if (s < 0) s = out[0];
  int e = behind ? i + 1 + __builtin_ctzll(behind) : S;
  for (int w = wid + 1; e == S && w < ST / 64; ++w) e = first[w];
  if (e == S) e = out[1];

  const I id = row[i];
  const long long n = (long long)B * S;
  int* y = spans + (long long)b * S + i;
  if (id < 0) {
    for (int k = 0; k < 4; ++k) y[k * n] = i;
    return;
  }
  int p = 0;
  if (prefix != nullptr && id < N) p = max(prefix[(long long)b * N + id], 0);
  p = min(p, e - s) + s;
  y[0] = s;
  y[n] = causal ? max(i + 1, p) : e;
  y[2 * n] = causal && i >= p ? i : s;
  y[3 * n] = e;
}

template <int D, int CAP, bool BIAS, int NW, int KB>
int launch_fwd(const Args& a, hipStream_t s) {
  const int blocks = (a.S + 32 * NW - 1) / (32 * NW), heads = a.B * a.H;
  hipLaunchKernelGGL((fwd_kernel<D, CAP, BIAS, NW, KB>),
                     dim3((unsigned)blocks * heads), dim3(64 * NW), 0, s, a,
                     blocks, heads);
  return (int)hipGetLastError();
}

template <int D, int CAP, bool BIAS>
int launch_bwd(const Args& a, int splits, hipStream_t s) {
  const int blocks = (a.S + 127) / 128;
  hipLaunchKernelGGL((dq_kernel<D, CAP, BIAS>),
                     dim3((unsigned)blocks * a.B * a.H), dim3(256), 0, s, a,
                     blocks, a.B * a.H);
  hipLaunchKernelGGL((dkdv_kernel<D, CAP, BIAS>),
                     dim3((unsigned)blocks * a.B * a.Hkv, splits), dim3(256),
                     0, s, a, blocks, a.B * a.Hkv);
  if (splits > 1) {
    const long long n = (long long)a.B * a.S * a.Hkv * D;
    hipLaunchKernelGGL(add_kernel, dim3((unsigned)((2 * n / 4 + 255) / 256)),
                       dim3(256), 0, s, a.part, a.dk, a.dv, n, splits, a.scale);
  }
  return (int)hipGetLastError();
}

template <int D>
int launch(const Args& a, int splits, hipStream_t s) {
  const bool bias = a.slopes != nullptr;
  // Steps of 32 keys leave room for three workgroups a CU where heads of 96 and 128
  // need registers for two otherwise (us, 64 / 32 keys: 1 x 8192 capped 811 / 769, nine
  // documents in 4 x 4096 258 / 230, heads of 96 273 / 250); heads of 64 hold four
  // either way (59 / 62). Eight waves that share the tiles took 883, 305, 296 and 64.
  constexpr int KB = D == 64 ? 64 : 32;
#define GO(C, W)                              \
  (splits ? launch_bwd<D, C, W>(a, splits, s) \
          : launch_fwd<D, C, W, 4, KB>(a, s))
  if (a.cap == 0.f) return bias ? GO(NONE, true) : GO(NONE, false);
  if (a.cap <= 200.f * LOG2E) return bias ? GO(USUAL, true) : GO(USUAL, false);
  return bias ? GO(WIDE, true) : GO(WIDE, false);
#undef GO
}

View view(const long long* s) { return View{s[0], s[1], s[2]}; }

}  // namespace

// ids [B, S] int32 (or int64, wide), prefix [B, N] or null, spans [4, B, S].
extern "C" int ds_packed_spans(const void* ids, int wide, const int* prefix,
                               int* spans, int B, int S, int N, int causal,
                               void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((S + ST - 1) / ST, B);
  if (wide)
    hipLaunchKernelGGL((spans_kernel<long long>), grid, dim3(ST), 0, s,
                       (const long long*)ids, prefix, spans, B, S, N, causal);
  else
    hipLaunchKernelGGL((spans_kernel<int>), grid, dim3(ST), 0, s,
                       (const int*)ids, prefix, spans, B, S, N, causal);
  return (int)hipGetLastError();
}

// splits 0: forward (out, lse and, unless null, rest written). Else backward from out,
// lse, rest and dout: dq, dk, dv contiguous, stat B H S floats, part splits 2 B S Hkv D
// (or null, 1).
// strides: (batch, token, head) of q, k, v, out, dout. cap 0: none. A hipError_t.
extern "C" int ds_masked_attention(
    const void* q, const void* k, const void* v, void* out, float* lse,
    void* rest, const void* dout, void* dq, void* dk, void* dv, float* stat,
    float* part, int splits, const int* spans, const float* slopes,
    const long long* strides, int B, int S, int H, int Hkv, int D, int causal,
    float scale, float cap, void* stream) {
  Args a;
  a.q = (const short*)q; a.k = (const short*)k; a.v = (const short*)v;
  a.o = (const short*)out; a.dout = (const short*)dout;
  a.out = (short*)out; a.dq = (short*)dq; a.dk = (short*)dk; a.dv = (short*)dv;
  a.lse = lse; a.rest = (int*)rest; a.stat = stat; a.part = splits > 1 ? part : nullptr;
  a.spans = spans; a.slopes = slopes;
  a.vq = view(strides); a.vk = view(strides + 3); a.vv = view(strides + 6);
  a.vo = view(strides + 9);
  a.vd = splits ? view(strides + 12) : View{0, 0, 0};
  a.B = B; a.S = S; a.H = H; a.Hkv = Hkv; a.causal = causal;
  a.scale = scale;
  a.c = scale * LOG2E;
  a.cap = cap * LOG2E;
  a.x = cap > 0.f ? scale / cap : 0.f;
  a.a = 2.f * LOG2E * a.x;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (D == 64) return launch<64>(a, splits, s);
  if (D == 96) return launch<96>(a, splits, s);
  return launch<128>(a, splits, s);
}
