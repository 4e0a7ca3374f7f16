// RMS norms of the queries' and keys' heads with the position rotation behind them,
// forward and backward, for MI355X (gfx950): what a layer does between its joint
// projection and its attention, in one launch.
//
//   n = x r w,  r = 1 / sqrt(mean x^2 + eps),  y = R(position) n
//   dn = R^T dy,  dw = sum dn x r,  dx = r (dn w - x r mean(dn w x r))
//
// A head is read once: a group of lanes holds it, two chunks of V coordinates a
// lane, chosen so that the pairs that turn together lie in one lane (`Places`). A
// wave stays with one token and takes its heads in turn, so that the angles are read
// once a token and not once a head. All in fp32, rounded once at the end. Bound by
// the stream of heads in and out: 8192 tokens, 32 and 8 heads of 128, bf16: 34 us forward
// (168 MB, 4.9 TB/s), 60 backward (252 MB, 4.2 TB/s) and 4 for the weights' sums; 100
// without the next heads' loads in flight. 16 tokens 4.6 us, a launch.

#include "ds_kernels.h"

namespace {

constexpr int CT = 256, NW = CT / 64;
constexpr int PARTS = 1024;       // workgroups of the backward: all resident at once

struct Heads {            // of q, then of k
  const void* x[2];
  void* y[2];             // contiguous
  const void* dy[2];      // backward
  const void* w[2];
  long long xb[2], xs[2], xh[2];      // strides of batch, token and head
  long long db[2], ds[2], dh[2];
  int heads[2];
};

struct Shape {
  const float* cs;        // [angles, rotated / 2]
  const float* sn;
  const int* positions;   // [tokens] or null: the token's place in S
  int tokens, S, D, rotated, angles;
  int per;                // lanes that hold a head
  int group;              // the same, up to a power of two
  float eps, plus;        // the weights' 1 + w
};

struct True { static constexpr bool value = true; };
struct False { static constexpr bool value = false; };

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// Where the two chunks of unit l of a head begin, and whether they turn. `half`: i
// turns with i + rotated / 2, and so do the chunks; else neighbours do.
template <int V>
struct Places {
  int a, b;
  bool turns;
  __device__ __forceinline__ Places(const Shape& s, bool half, int l) {
    const int n = s.rotated / (2 * V);
    turns = l < n;
    if (half && turns) {
      a = l * V;
      b = s.rotated / 2 + l * V;
    } else {
      a = 2 * V * l;
      b = a + V;
    }
  }
};

// Both chunks' coordinates turned by the lane's V angles (sign -1: back).
template <int V, bool HALF>
__device__ __forceinline__ void turn(float (&z)[2 * V], const float (&c)[V],
                                     const float (&s)[V], float sign) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int i = HALF || V == 1 ? e : 2 * e;
    const int j = HALF || V == 1 ? e + V : 2 * e + 1;
    const ds::Turned t = ds::turn(z[i], z[j], c[e], sign * s[e]);
    z[i] = t.lo;
    z[j] = t.hi;
  }
}

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, int a, int b,
                                     float (&z)[2 * V]) {
  const Vec<T, V> x = *(const Vec<T, V>*)(p + a), y = *(const Vec<T, V>*)(p + b);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    z[e] = ds::to_f32(x.v[e]);
    z[V + e] = ds::to_f32(y.v[e]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, int a, int b,
                                      const float (&z)[2 * V]) {
  Vec<T, V> x, y;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    x.v[e] = ds::from_f32<T>(z[e]);
    y.v[e] = ds::from_f32<T>(z[V + e]);
  }
  *(Vec<T, V>*)(p + a) = x;
  *(Vec<T, V>*)(p + b) = y;
}

// A token's angles for the lane's units; no position, no numbers.
template <int V, int R>
__device__ __forceinline__ void angles(const Shape& s, int token, int sub,
                                       float (&c)[R][V], float (&sn)[R][V],
                                       float& fault) {
  const int pos = s.positions ? s.positions[token] : token % s.S;
  const bool there = pos >= 0 && pos < s.angles;
  fault = there ? 0.f : __builtin_nanf("");
  const long long at = (long long)(there ? pos : 0) * (s.rotated / 2);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int l = sub + r * 64;
    const bool turns = l < s.rotated / (2 * V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[r][e] = turns ? s.cs[at + l * V + e] : 1.f;
      sn[r][e] = turns ? s.sn[at + l * V + e] : 0.f;
    }
  }
}

__device__ __forceinline__ float group_sum(float x, int group) {
  for (int off = group >> 1; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// Workgroup (x, y): tokens 4 x .. 4 x + 3, a wave each; y: a share of the heads. The
// next heads are in flight behind these ones' arithmetic.
template <typename T, int V, int R, bool HALF>
__global__ __launch_bounds__(CT) void fwd_kernel(const Heads p,
                                                 const Shape s) {
  const int lane = threadIdx.x & 63;
  const int token = blockIdx.x * NW +
                    __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (token >= s.tokens) return;
  const int sub = lane & (s.group - 1), g = lane / s.group;
  const int at_once = 64 / s.group, all = p.heads[0] + p.heads[1];
  const long long b = token / s.S, t = token % s.S;
  Vec<T, V> next[R][2];
  auto fetch = [&](int h0) __attribute__((always_inline)) {
    int h = min(h0 + g, all - 1);
    const int k = h >= p.heads[0];
    if (k) h -= p.heads[0];
    const T* x = (const T*)p.x[k] + b * p.xb[k] + t * p.xs[k] + h * p.xh[k];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Places<V> at(s, HALF, sub + r * 64);
      if (sub + r * 64 < s.per) {
        next[r][0] = *(const Vec<T, V>*)(x + at.a);
        next[r][1] = *(const Vec<T, V>*)(x + at.b);
      }
    }
  };
  const int step = gridDim.y * at_once;
  if ((int)blockIdx.y * at_once < all) fetch(blockIdx.y * at_once);
  float c[R][V], sn[R][V], fault;
  angles<V, R>(s, token, sub, c, sn, fault);
  for (int h0 = blockIdx.y * at_once; h0 < all; h0 += step) {
    float z[R][2 * V], sum = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (sub + r * 64 < s.per)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          z[r][e] = ds::to_f32(next[r][0].v[e]);
          z[r][V + e] = ds::to_f32(next[r][1].v[e]);
          sum += z[r][e] * z[r][e] + z[r][V + e] * z[r][V + e];
        }
    if (h0 + step < all) fetch(h0 + step);
    sum = group_sum(sum, s.group);
    const float scale = 1.f / sqrtf(sum / s.D + s.eps) + fault;
    int h = h0 + g;
    if (h >= all) continue;
    const int k = h >= p.heads[0];
    if (k) h -= p.heads[0];
    T* y = (T*)p.y[k] + ((long long)token * p.heads[k] + h) * s.D;
    const T* w = (const T*)p.w[k];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Places<V> at(s, HALF, sub + r * 64);
      if (sub + r * 64 < s.per) {
        float wf[2 * V];
        load<T, V>(w, at.a, at.b, wf);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) z[r][e] *= scale * (wf[e] + s.plus);
        if (at.turns) turn<V, HALF>(z[r], c[r], sn[r], 1.f);
        store<T, V>(y, at.a, at.b, z[r]);
      }
    }
  }
}

// Backward: workgroups of queries (the first `first`) and of keys, so that a lane keeps
// the sums of one weight's gradient. Every wave goes through an even share of the
// rounds, some heads of a token each (or all heads of some tokens, where they are few),
// one token's behind another's, the next round's heads in flight behind this one's
// arithmetic. Tokens are counted by the scalar unit: with every group on a head of its
// own, wherever it is, 8192 tokens of 32 and 8 heads of 128 took 79 us for 60. part [workgroups][D], added up in their
// order by sum_kernel.
template <typename T, int V, int R, bool HALF>
__global__ __launch_bounds__(CT, 4) void bwd_kernel(const Heads p, const Shape s,
                                                 float* __restrict__ part,
                                                 const int first) {
  extern __shared__ float lds[];       // [NW][D]
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = lane & (s.group - 1), g = lane / s.group;
  const int at_once = 64 / s.group;
  const int k = (int)blockIdx.x >= first;
  const int all = p.heads[k];
  const int blocks = k ? gridDim.x - first : first;
  const long long wave = ((long long)blockIdx.x - (k ? first : 0)) * NW + wid;
  const int rounds = (all + at_once - 1) / at_once;    // of a token
  const int span = all < at_once ? at_once / all : 1;  // tokens of a round
  const int more = span > 1 ? g / all : 0, first_head = span > 1 ? g % all : g;
  const bool spare = more >= span;                     // the group has no head
  const long long total =
      (long long)((s.tokens + span - 1) / span) * rounds;
  const int waves = blocks * NW;
  const long long begin = total * wave / waves, end = total * (wave + 1) / waves;

  float w[R][2 * V], dw[R][2 * V] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Places<V> at(s, HALF, sub + r * 64);
    if (sub + r * 64 < s.per) {
      load<T, V>((const T*)p.w[k], at.a, at.b, w[r]);
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) w[r][e] += s.plus;
    }
  }
  struct Raw {
    Vec<T, V> x[R][2], d[R][2];
  };
  auto run = [&](auto many) __attribute__((always_inline)) {
    constexpr bool MANY = decltype(many)::value;
    int token = (int)(begin / rounds) * (MANY ? span : 1), round = (int)(begin % rounds);
    // where there is none, the last
    auto own = [&]() { return min(token + more, s.tokens - 1); };
    auto fetch = [&](Raw& raw) __attribute__((always_inline)) {
      const int h = min(round * at_once + first_head, all - 1);
      long long b = token / s.S, t = token % s.S;
      if (MANY) {
        b = own() / s.S;
        t = own() % s.S;
      }
      const T* x = (const T*)p.x[k] + b * p.xb[k] + t * p.xs[k] + h * p.xh[k];
      const T* d = (const T*)p.dy[k] + b * p.db[k] + t * p.ds[k] + h * p.dh[k];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Places<V> at(s, HALF, sub + r * 64);
        if (sub + r * 64 < s.per) {
          raw.x[r][0] = *(const Vec<T, V>*)(x + at.a);
          raw.x[r][1] = *(const Vec<T, V>*)(x + at.b);
          raw.d[r][0] = *(const Vec<T, V>*)(d + at.a);
          raw.d[r][1] = *(const Vec<T, V>*)(d + at.b);
        }
      }
    };
    Raw next;
    if (begin < end) fetch(next);
    int known = -1;
    float c[R][V], sn[R][V], fault = 0.f;
    for (long long i = begin; i < end; ++i) {
      if (token != known)
        angles<V, R>(s, MANY ? own() : token, sub, c, sn, fault);
      known = token;
      float z[R][2 * V], d[R][2 * V], sum = 0.f, mix = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          z[r][e] = ds::to_f32(next.x[r][0].v[e]);
          z[r][V + e] = ds::to_f32(next.x[r][1].v[e]);
          d[r][e] = ds::to_f32(next.d[r][0].v[e]);
          d[r][V + e] = ds::to_f32(next.d[r][1].v[e]);
        }
      const int here = MANY ? token + more : token, h = round * at_once + first_head;
      const bool live = h < all && (!MANY || (!spare && here < s.tokens));
      if (++round == rounds) {
        round = 0;
        token += MANY ? span : 1;
      }
      if (i + 1 < end) fetch(next);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Places<V> at(s, HALF, sub + r * 64);
        if (sub + r * 64 < s.per) {
          if (at.turns) turn<V, HALF>(d[r], c[r], sn[r], -1.f);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) {
            sum += z[r][e] * z[r][e];
            mix += d[r][e] * w[r][e] * z[r][e];
          }
        }
      }
      sum = group_sum(sum, s.group);
      mix = group_sum(mix, s.group);
      const float scale = 1.f / sqrtf(sum / s.D + s.eps) + fault;
      const float back = mix * scale * scale / s.D;      // of x
      if (!live) continue;
      T* dx = (T*)p.y[k] + ((long long)here * all + h) * s.D;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Places<V> at(s, HALF, sub + r * 64);
        if (sub + r * 64 < s.per) {
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) {
            dw[r][e] += d[r][e] * z[r][e] * scale;
            d[r][e] = scale * (d[r][e] * w[r][e] - z[r][e] * back);
          }
          store<T, V>(dx, at.a, at.b, d[r]);
        }
      }
    }
  };
  if (span > 1) run(True());
  else run(False());
  // the groups of a wave, then the waves
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Places<V> at(s, HALF, sub + r * 64);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) {
      float u = dw[r][e];
      for (int off = s.group; off < 64; off <<= 1) u += __shfl_xor(u, off, 64);
      if (g == 0 && sub + r * 64 < s.per)
        lds[wid * s.D + (e < V ? at.a + e : at.b + e - V)] = u;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s.D; i += CT) {
    float u = 0.f;
#pragma unroll
    for (int n = 0; n < NW; ++n) u += lds[n * s.D + i];
    part[(long long)blockIdx.x * s.D + i] = u;
  }
}

// dq from part [first][D], dk from the rows behind: 8 columns a workgroup, 32 threads a
// column.
template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(
    const float* __restrict__ part, T* __restrict__ dq, T* __restrict__ dk,
    const int first, const int n, const int D) {
  __shared__ float lds[32][9];
  const int col = threadIdx.x & 7, row = threadIdx.x >> 3;
  const int i = blockIdx.x * 8 + col;
  const int k = i >= D, lo = k ? first : 0, hi = k ? n : first;
  float u = 0.f;
  if (i < 2 * D)
#pragma unroll 8
    for (int r = lo + row; r < hi; r += 32)
      u += part[(long long)r * D + (k ? i - D : i)];
  lds[row][col] = u;
  __syncthreads();
  if (row == 0 && i < 2 * D) {
    for (int r = 1; r < 32; ++r) u += lds[r][col];
    (k ? dk + i - D : dq + i)[0] = ds::from_f32<T>(u);
  }
}

template <typename T, int V, int R>
int launch(const Heads& p, const Shape& s, bool half, float* part, int parts,
           void* dqw, void* dkw, hipStream_t st) {
  const int at_once = 64 / s.group, all = p.heads[0] + p.heads[1];
  if (part == nullptr) {
    // few tokens: their heads spread over as many waves as there are
    int shares = 1;
    const int rounds = (all + at_once - 1) / at_once;
    while (shares < rounds && (long long)s.tokens * shares < 2048) ++shares;
    const dim3 grid((s.tokens + NW - 1) / NW, shares);
    if (half)
      hipLaunchKernelGGL((fwd_kernel<T, V, R, true>), grid, dim3(CT), 0, st, p,
                         s);
    else
      hipLaunchKernelGGL((fwd_kernel<T, V, R, false>), grid, dim3(CT), 0, st, p,
                         s);
    return (int)hipGetLastError();
  }
  const int lds = NW * s.D * sizeof(float);
  // workgroups by rounds, but some for both
  auto rounds = [&](int heads) {
    return heads < at_once ? 1.0 / (at_once / heads)
                           : (double)((heads + at_once - 1) / at_once);
  };
  const double q = rounds(p.heads[0]), k = rounds(p.heads[1]);
  int first = (int)(parts * q / (q + k) + 0.5);
  first = first < 1 ? 1 : first > parts - 1 ? parts - 1 : first;
  if (half)
    hipLaunchKernelGGL((bwd_kernel<T, V, R, true>), dim3(parts), dim3(CT), lds,
                       st, p, s, part, first);
  else
    hipLaunchKernelGGL((bwd_kernel<T, V, R, false>), dim3(parts), dim3(CT), lds,
                       st, p, s, part, first);
  hipLaunchKernelGGL((sum_kernel<T>), dim3((2 * s.D + 7) / 8), dim3(256), 0, st,
                     part, (T*)dqw, (T*)dkw, first, parts, s.D);
  return (int)hipGetLastError();
}

}  // namespace

// Workgroups of the backward, each of which leaves [D] floats: of queries and of keys.
extern "C" int ds_qk_norm_parts(int tokens) {
  const int n = 2 * ((tokens + NW - 1) / NW);
  return n < PARTS ? n : PARTS;
}

// Forward: x to y. Backward (part given): dy and x to y, and the weights' gradients.
// strides: (batch, token, head) of q, k, and of dq, dk. type: 0 fp32, 1 bf16, 2
// fp16. Even D up to 512 and even rotated up to D. A hipError_t, or -1.
extern "C" int ds_qk_norm_rope(
    const void* q, const void* k, void* yq, void* yk, const void* dq,
    const void* dk, const void* wq, const void* wk, const float* cs,
    const float* sn, const int* positions, const long long* strides, int B,
    int S, int H, int Hk, int D, int rotated, int angles, int half, float eps,
    float plus, int type, float* part, int parts, void* dwq, void* dwk,
    void* stream) {
  if (D < 2 || D > 512 || D % 2 || rotated < 2 || rotated > D || rotated % 2)
    return -1;
  const bool back = part != nullptr;
  Heads p = {{q, k}, {yq, yk}, {dq, dk}, {wq, wk}, {}, {}, {}, {}, {}, {},
             {H, Hk}};
  const int size = type == 0 ? 4 : 2;
  // the largest chunk that every row, weight and pair allows
  int V = 16 / size;
  auto fits = [&](int v) {
    const int bytes = v * size;
    if (half ? rotated / 2 % v || (D - rotated) % (2 * v)
             : rotated % (2 * v) || D % (2 * v))
      return false;
    for (const void* x : {q, k, (const void*)yq, (const void*)yk, dq, dk, wq, wk})
      if ((uintptr_t)x % bytes) return false;
    for (int i = 0; i < (back ? 12 : 6); ++i)
      if (strides[i] % v) return false;
    return true;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  for (int i = 0; i < 2; ++i) {
    p.xb[i] = strides[3 * i];
    p.xs[i] = strides[3 * i + 1];
    p.xh[i] = strides[3 * i + 2];
    if (back) {
      p.db[i] = strides[6 + 3 * i];
      p.ds[i] = strides[6 + 3 * i + 1];
      p.dh[i] = strides[6 + 3 * i + 2];
    }
  }
  Shape s = {cs, sn, positions, B * S, S, D, rotated, angles, D / (2 * V), 1,
             eps, plus};
  while (s.group < s.per && s.group < 64) s.group <<= 1;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define GO(T, V_)                                                             \
  if constexpr (V_ <= 2)      /* heads of up to 512 in at most 64 lanes */    \
    if (s.per > 64)                                                           \
      return launch<T, V_, 4 / V_>(p, s, half, part, parts, dwq, dwk, st);    \
  return launch<T, V_, 1>(p, s, half, part, parts, dwq, dwk, st)
#define TYPE(T)            \
  if (V == 4) { GO(T, 4); } \
  if (V == 2) { GO(T, 2); } \
  GO(T, 1)
  if (type == 0) { TYPE(float); }
  if (type == 1) {
    if (V == 8) { GO(ds::bf16, 8); }
    TYPE(ds::bf16);
  }
  if (V == 8) { GO(ds::f16, 8); }
  TYPE(ds::f16);
#undef TYPE
#undef GO
}
