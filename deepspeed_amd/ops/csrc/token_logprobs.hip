// Log probabilities of given tokens, with the entropy of their distribution and its
// best tokens, for MI355X (gfx950). logits [N, V] fp32, bf16 or fp16.
//
//   m = max x, s = sum e^(x - m), u = sum e^(x - m) (x - m)
//   logprob = x_y - m - log s,  entropy = log s - u / s
//   dx_j = -p_j (g + h (x_j - m - log s + entropy)) + [j = y] g,  p_j = e^(x_j - m) / s
//
// for the gradients g of the log probability and h of the entropy. All sums are
// fp32, of differences to the maximum, so that large logits cost no digits; x - m is
// taken before it is scaled to a power of two for the same reason.
//
// Bound by the logits' stream: read once forward, read and written once backward.

#include "ds_kernels.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3.0e38f;     // a maximum before anything was seen
constexpr int CT = 256;                // threads of a workgroup
constexpr int HELD = 32;               // logits that a thread holds
constexpr int PART = CT * HELD;        // logits of a part of a row

template <typename T>
struct alignas(16) Chunk {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Rows of logits: row r is row r % inner of r / inner.
struct Rows {
  const void* x;
  long long outer_stride, inner_stride;
  int inner;
  __device__ __forceinline__ long long at(int r) const {
    return r / inner * outer_stride + r % inner * inner_stride;
  }
};

__device__ __forceinline__ float power(float d2) {
  return __builtin_amdgcn_exp2f(d2);
}

struct Sums {
  float m = LOWEST, s = 0.f, u = 0.f;     // u in units of log2
  __device__ __forceinline__ void raise(float t) {
    if (t > m) {
      const float d2 = (m - t) * LOG2E;
      const float f = power(d2);
      // of nothing seen yet, d2 is as good as -inf
      u = s > 0.f ? f * __builtin_fmaf(s, d2, u) : 0.f;
      s *= f;
      m = t;
    }
  }
  __device__ __forceinline__ void add(float x) {
    const float d2 = (x - m) * LOG2E, e = power(d2);
    s += e;
    u = __builtin_fmaf(e, d2, u);
  }
  // an infinite logit has no share, where its product would be no number
  __device__ __forceinline__ void add_any(float x) {
    const float d2 = (x - m) * LOG2E, e = power(d2);
    s += e;
    u = __builtin_fmaf(e, fmaxf(d2, -1e30f), u);
  }
};

// Over the 64 lanes by moves inside the vector unit: rows of 16, the rows of a half,
// the halves; the last lane has it all. Six exchanges through LDS take as long as
// thirty of these, and a best token takes one or two such reductions.
template <typename Op>
__device__ __forceinline__ int over_lanes(int x, int none, Op op) {
#define STEP(CTRL, ROWS) \
  x = op(x, __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false))
  STEP(0x111, 0xf);      // one lane up, two, four, eight
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);      // a row's last lane to the next row
  STEP(0x143, 0xc);      // the first half's to the second
#undef STEP
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ float as_float(int x) {
  return __builtin_bit_cast(float, x);
}
__device__ __forceinline__ int as_int(float x) {
  return __builtin_bit_cast(int, x);
}
__device__ __forceinline__ float lanes_max(float x) {
  return as_float(over_lanes(as_int(x), as_int(LOWEST), [](int a, int b) {
    return as_int(fmaxf(as_float(a), as_float(b)));
  }));
}
__device__ __forceinline__ float lanes_sum(float x) {
  return as_float(over_lanes(as_int(x), 0, [](int a, int b) {
    return as_int(as_float(a) + as_float(b));
  }));
}

// The lanes' sums as if one lane had seen all.
__device__ __forceinline__ void join_lanes(Sums& a) {
  const float m = lanes_max(a.m);
  const float d2 = (a.m - m) * LOG2E, f = power(d2);
  float u = a.s > 0.f ? f * __builtin_fmaf(a.s, d2, a.u) : 0.f;
  float s = a.s * f;
  if (a.s != a.s) s = u = a.s;
  a.s = lanes_sum(s);
  a.u = lanes_sum(u);
  a.m = m;
}
__device__ __forceinline__ void join_waves(Sums& a, float (*lds)[3]) {
  join_lanes(a);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) {
    lds[wid][0] = a.m;
    lds[wid][1] = a.s;
    lds[wid][2] = a.u;
  }
  __syncthreads();
  Sums w;
  if (lane < CT / 64) {
    w.m = lds[lane][0];
    w.s = lds[lane][1];
    w.u = lds[lane][2];
  }
  join_lanes(w);
  a = w;
}

// What a row comes to. A token outside of the row has no log probability.
__device__ __forceinline__ void finish(const Sums& a, float xy, bool known,
                                       float* lp, float* ent, float* stat) {
  const float logs = __builtin_amdgcn_logf(a.s);       // log2
  *lp = known ? ((xy - a.m) * LOG2E - logs) * LN2 : __builtin_nanf("");
  *ent = (logs - a.u / a.s) * LN2;
  stat[0] = a.m;
  stat[1] = logs;
}

// ------------------------------------------------- many rows: a workgroup each

template <typename T>
__global__ __launch_bounds__(CT) void rows_kernel(
    const Rows rows, const long long* __restrict__ tokens,
    float* __restrict__ lp, float* __restrict__ ent, float* __restrict__ stat,
    const long long V, const long long ignore) {
  constexpr int N = Chunk<T>::N, U = 4;
  __shared__ float lds[CT / 64][3];
  const int row = blockIdx.x, tid = threadIdx.x;
  const long long y = tokens[row];
  if (y == ignore) {
    if (tid == 0) {
      lp[row] = ent[row] = 0.f;
      stat[2 * row] = stat[2 * row + 1] = 0.f;
    }
    return;
  }
  const T* x = (const T*)rows.x + rows.at(row);
  const long long head =
      min((long long)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), V);
  const long long nv = (V - head) / N;
  const Chunk<T>* xv = (const Chunk<T>*)(x + head);

  Sums a;
  auto one = [&](float v, bool any) {
    a.raise(v);
    any ? a.add_any(v) : a.add(v);
  };
  auto pass = [&](bool any) __attribute__((always_inline)) {
    a = Sums();
    for (long long j = tid; j < head; j += CT) one(ds::to_f32(x[j]), any);
    long long j = tid;
    for (; j + (U - 1) * CT < nv; j += U * CT) {
      Chunk<T> v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = xv[j + i * CT];
      float t = LOWEST;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) t = fmaxf(t, ds::to_f32(v[i].v[e]));
      a.raise(t);
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
          any ? a.add_any(ds::to_f32(v[i].v[e])) : a.add(ds::to_f32(v[i].v[e]));
    }
    for (; j < nv; j += CT) {
      const Chunk<T> v = xv[j];
#pragma unroll
      for (int e = 0; e < N; ++e) one(ds::to_f32(v.v[e]), any);
    }
    for (long long k = head + nv * N + tid; k < V; k += CT)
      one(ds::to_f32(x[k]), any);
    join_waves(a, lds);
  };
  pass(false);
  // infinite logits among others: once more, with care
  if (a.u != a.u && a.s == a.s) pass(true);
  if (tid == 0) {
    const bool known = y >= 0 && y < V;
    finish(a, known ? ds::to_f32(x[y]) : 0.f, known, lp + row, ent + row,
           stat + 2 * row);
  }
}

// ------------------------------------------- few rows, or their best tokens too
//
// Parts of 8192 logits, held in registers: the sums of each, and of each wave its
// best, sorted. join_kernel makes a row of the parts.

struct Best {
  unsigned key;     // grows with the logit, NaN above all
  int id;
};

__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);   // -0 is 0
  return x != x ? ~0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
  return key == ~0u ? __builtin_nanf("")
                    : __builtin_bit_cast(
                          float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The lane whose key is the largest, of equal ones the lowest id.
__device__ __forceinline__ int best_lane(unsigned key, int id) {
  const int top = over_lanes((int)key, 0, [](int a, int b) {
    return (int)max((unsigned)a, (unsigned)b);
  });
  unsigned long long who = __ballot(key == (unsigned)top);
  if (who & (who - 1)) {
    const int low = over_lanes(key == (unsigned)top ? id : 0x7fffffff,
                               0x7fffffff,
                               [](int a, int b) { return min(a, b); });
    who = __ballot(key == (unsigned)top && id == low);
  }
  return __builtin_ctzll(who);
}

template <typename T>
__global__ __launch_bounds__(CT) void parts_kernel(
    const Rows rows, const long long* __restrict__ tokens,
    float* __restrict__ sums,          // [N, parts, 3]
    Best* __restrict__ lists,          // [N, parts, waves, top]
    const long long V, const int parts, const int top,
    const long long ignore) {
  constexpr int N = Chunk<T>::N, C = HELD / N;
  __shared__ float lds[CT / 64][3];
  const int row = blockIdx.x / parts, part = blockIdx.x % parts;
  const int tid = threadIdx.x;
  const int lane = tid & 63, wid = tid >> 6;
  if (tokens[row] == ignore) return;
  const T* x = (const T*)rows.x + rows.at(row);
  // chunks lie on 16 bytes: the first and the last may reach out of the row
  const int ahead = (int)(((uintptr_t)x & 15) / sizeof(T));
  const long long first = (long long)part * PART + tid * N - ahead;
  float v[HELD];
  unsigned gone = 0;                   // places that are none
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const long long j = first + (long long)c * CT * N;
    if (j >= 0 && j + N <= V) {
      const Chunk<T> y = *(const Chunk<T>*)(x + j);
#pragma unroll
      for (int e = 0; e < N; ++e) v[c * N + e] = ds::to_f32(y.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool in = j + e >= 0 && j + e < V;
        v[c * N + e] = in ? ds::to_f32(x[j + e]) : -__builtin_inff();
        if (!in) gone |= 1u << (c * N + e);
      }
    }
  }
  Sums a;
#pragma unroll
  for (int e = 0; e < HELD; ++e) a.m = fmaxf(a.m, v[e]);
#pragma unroll
  for (int e = 0; e < HELD; ++e) a.add_any(v[e]);
  join_waves(a, lds);
  if (tid == 0) {
    float* s = sums + ((long long)row * parts + part) * 3;
    s[0] = a.m;
    s[1] = a.s;
    s[2] = a.u;
  }
  Best* list =
      lists + (((long long)row * parts + part) * (CT / 64) + wid) * top;
  if (top == 0) return;
  unsigned keys[HELD], key = 0;
#pragma unroll
  for (int e = 0; e < HELD; ++e) keys[e] = gone >> e & 1 ? 0u : key_of(v[e]);
  int place = -1;
  // the lane's best but for `place`, which was taken
  auto look = [&]() __attribute__((always_inline)) {
    const int taken = place;
    key = 0;
    place = 0;
#pragma unroll
    for (int e = 0; e < HELD; ++e) {
      if (e == taken) keys[e] = 0;
      if (keys[e] > key) {
        key = keys[e];
        place = e;
      }
    }
  };
  look();
  for (int i = 0; i < top; ++i) {
    const int id =
        (int)(first + (long long)(place / N) * CT * N + place % N);
    const int who = best_lane(key, id);
    if (lane == who) {
      list[i] = Best{key, id};         // key 0: the wave has no more
      look();
    }
  }
}

// A wave a row. Its lists are in LDS, lane l looks after the lists l, l + 64 ...
__global__ __launch_bounds__(64) void join_kernel(
    const Rows rows, const int type, const long long* __restrict__ tokens,
    const float* __restrict__ sums, const Best* __restrict__ lists,
    float* __restrict__ lp, float* __restrict__ ent, float* __restrict__ stat,
    float* __restrict__ top_lp, long long* __restrict__ top_ids,
    const long long V, const int parts, const int top,
    const long long ignore) {
  extern __shared__ Best held[];
  const int row = blockIdx.x, lane = threadIdx.x;
  const long long y = tokens[row];
  const long long out = (long long)row * top;
  if (y == ignore) {
    if (lane == 0) {
      lp[row] = ent[row] = 0.f;
      stat[2 * row] = stat[2 * row + 1] = 0.f;
    }
    if (lane < top) {
      top_lp[out + lane] = -__builtin_inff();
      top_ids[out + lane] = -1;
    }
    return;
  }
  const int n = parts * (CT / 64);
  const Best* from = lists + (long long)row * n * top;
  for (int i = lane; i < n * top; i += 64) held[i] = from[i];
  Sums a;
  for (int i = lane; i < parts; i += 64) {
    const float* p = sums + ((long long)row * parts + i) * 3;
    Sums b;
    b.m = p[0]; b.s = p[1]; b.u = p[2];
    const float m = fmaxf(a.m, b.m);
    a.raise(m);
    b.raise(m);
    a.s += b.s;
    a.u += b.u;
  }
  join_lanes(a);
  const float logs = __builtin_amdgcn_logf(a.s);
  if (lane == 0) {
    const bool known = y >= 0 && y < V;
    const long long at = rows.at(row) + (known ? y : 0);
    const float xy = type == 0   ? ((const float*)rows.x)[at]
                     : type == 1 ? ds::to_f32(((const ds::bf16*)rows.x)[at])
                                 : ds::to_f32(((const ds::f16*)rows.x)[at]);
    finish(a, xy, known, lp + row, ent + row, stat + 2 * row);
  }
  __syncthreads();
  // of each of the lane's lists the next one to look at
  int next[4] = {0, 0, 0, 0}, mine = 0;
  Best b;
  auto look = [&]() __attribute__((always_inline)) {
    b = Best{0u, 0x7fffffff};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int l = lane + 64 * u;
      if (l < n && next[u] < top) {
        const Best c = held[l * top + next[u]];
        if (c.key > b.key || (c.key == b.key && c.id < b.id)) {
          b = c;
          mine = u;
        }
      }
    }
  };
  if (top) look();
  for (int i = 0; i < top; ++i) {
    if (lane == best_lane(b.key, b.id)) {
      top_lp[out + i] = ((logit_of(b.key) - a.m) * LOG2E - logs) * LN2;
      top_ids[out + i] = b.id;
#pragma unroll
      for (int u = 0; u < 4; ++u) next[u] += mine == u;
      look();
    }
  }
}

// ----------------------------------------------------------------- backward
//
// A workgroup a row, or a part of `span` logits of it where there are few rows.

template <typename T>
__global__ __launch_bounds__(CT) void grad_kernel(
    const Rows rows, const long long* __restrict__ tokens,
    const float* __restrict__ stat, const float* __restrict__ ent,
    const float* __restrict__ glp, const float* __restrict__ gent,
    T* __restrict__ dx, const long long V, const long long span,
    const long long ignore) {
  constexpr int N = Chunk<T>::N;
  const int row = blockIdx.x, tid = threadIdx.x;
  const long long y = tokens[row];
  const bool live = y != ignore;
  const long long lo = blockIdx.y * span, hi = min(V, lo + span);
  const T* x = (const T*)rows.x + rows.at(row);
  T* d = dx + (long long)row * V;
  const float m = stat[2 * row], logs = stat[2 * row + 1];
  float g = glp ? glp[row] : 0.f;
  if (y < 0 || y >= V) g = __builtin_nanf("");
  const float h = gent ? gent[row] : 0.f;
  // g + h (x - m - log s + entropy) = base + h ln 2 (d2), d2 as below
  const float slope = h * LN2, base = __builtin_fmaf(h, ent[row], g);
  auto one = [&](float v, long long j) -> T {
    const float d2 = (v - m) * LOG2E - logs, p = power(d2);
    // without a share none of the gradient either
    const float t = p == 0.f ? 0.f : -p * __builtin_fmaf(slope, d2, base);
    return ds::from_f32<T>(live ? (j == y ? t + g : t) : 0.f);
  };
  const bool same = (((uintptr_t)x ^ (uintptr_t)d) & 15) == 0;
  const long long head =
      same ? min((long long)((16 - ((uintptr_t)(x + lo) & 15)) & 15) /
                     (int)sizeof(T), hi - lo)
           : hi - lo;
  const long long nv = (hi - lo - head) / N, from = lo + head;
  for (long long j = lo + tid; j < from; j += CT)
    d[j] = one(ds::to_f32(x[j]), j);
  for (long long j = tid; j < nv; j += CT) {
    Chunk<T> v = *(const Chunk<T>*)(x + from + j * N);
#pragma unroll
    for (int e = 0; e < N; ++e)
      v.v[e] = one(ds::to_f32(v.v[e]), from + j * N + e);
    *(Chunk<T>*)(d + from + j * N) = v;
  }
  for (long long j = from + nv * N + tid; j < hi; j += CT)
    d[j] = one(ds::to_f32(x[j]), j);
}

}  // namespace

// Parts a row is cut into; 0: a workgroup a row.
extern "C" int ds_logprobs_parts(int rows, long long V, int top) {
  const long long parts = (V + PART + 6) / PART;   // a row may begin inside a chunk
  return top == 0 && (parts == 1 || rows >= 512) ? 0 : (int)parts;
}

// type: 0 fp32, 1 bf16, 2 fp16. parts as ds_logprobs_parts says, sums [N, parts, 3],
// lists [N, parts, 4, top] of 8 bytes. Returns a hipError_t.
extern "C" int ds_logprobs_fwd(const void* x, long long outer_stride,
                               long long inner_stride, int inner, int type,
                               const long long* tokens, float* lp, float* ent,
                               float* stat, float* top_lp, long long* top_ids,
                               float* sums, void* lists, int rows, long long V,
                               int parts, int top, long long ignore,
                               void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Rows r = {x, outer_stride, inner_stride, inner};
#define GO(T)                                                                  \
  if (parts == 0)                                                              \
    hipLaunchKernelGGL((rows_kernel<T>), dim3(rows), dim3(CT), 0, s, r,        \
                       tokens, lp, ent, stat, V, ignore);                      \
  else                                                                         \
    hipLaunchKernelGGL((parts_kernel<T>), dim3(parts * rows), dim3(CT), 0, s,  \
                       r, tokens, sums, (Best*)lists, V, parts, top, ignore)
  if (type == 0) { GO(float); }
  else if (type == 1) { GO(ds::bf16); }
  else { GO(ds::f16); }
#undef GO
  if (parts)
    hipLaunchKernelGGL(join_kernel, dim3(rows), dim3(64),
                       parts * (CT / 64) * top * sizeof(Best), s, r, type,
                       tokens, sums, (const Best*)lists, lp, ent, stat, top_lp,
                       top_ids, V, parts, top, ignore);
  return (int)hipGetLastError();
}

// dx [N, V] contiguous; glp and gent [N] or null.
extern "C" int ds_logprobs_bwd(const void* x, long long outer_stride,
                               long long inner_stride, int inner, int type,
                               const long long* tokens, const float* stat,
                               const float* ent, const float* glp,
                               const float* gent, void* dx, int rows,
                               long long V, long long ignore, void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Rows r = {x, outer_stride, inner_stride, inner};
  // whole rows from 2048 on; fewer are cut, but not below 4096 logits
  long long cuts = rows >= 2048 ? 1 : (2048 + rows - 1) / rows;
  if (cuts > (V + 4095) / 4096) cuts = (V + 4095) / 4096;
  const long long span = ((V + cuts - 1) / cuts + 7) / 8 * 8;
  const dim3 grid(rows, (unsigned)((V + span - 1) / span));
#define GO(T)                                                                 \
  hipLaunchKernelGGL((grad_kernel<T>), grid, dim3(CT), 0, s, r, tokens, stat, \
                     ent, glp, gent, (T*)dx, V, span, ignore)
  if (type == 0) GO(float);
  else if (type == 1) GO(ds::bf16);
  else GO(ds::f16);
#undef GO
  return (int)hipGetLastError();
}
