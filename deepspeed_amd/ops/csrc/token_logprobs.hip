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
// Bound by the logits' stream, read once forward, read and written once backward, past
// the caches, which they do not fit. 4096 x 128256 bf16: 154 us forward (6.8 TB/s; 199
// through the caches), masked or not, 411 backward (5.1 TB/s, a copy's rate).

#include "ds_kernels.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// A maximum before anything was seen: no finite logit lies below it.
constexpr float LOWEST = -__FLT_MAX__;
constexpr int CT = 256;                // threads of a workgroup
constexpr int HELD = 32;               // logits that a thread holds
constexpr int PART = CT * HELD;        // logits of a part of a row

template <typename T>
struct alignas(16) Chunk {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// A chunk that is read, or written, once: past the caches.
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Chunk<T> stream(const Chunk<T>* p) {
  return __builtin_bit_cast(Chunk<T>,
                            __builtin_nontemporal_load((const i32x4*)p));
}
template <typename T>
__device__ __forceinline__ void stream(Chunk<T>* p, const Chunk<T>& x) {
  __builtin_nontemporal_store(__builtin_bit_cast(i32x4, x), (i32x4*)p);
}

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
      // what has no share beside t adds nothing: s d2 may be past all numbers
      u = f > 0.f ? f * __builtin_fmaf(s, d2, u) : 0.f;
      s *= f;
      m = t;
    }
  }
  // an infinite logit, or one as far, has no share, where its product would be no number
  __device__ __forceinline__ void add(float x) {
    const float d2 = (x - m) * LOG2E, e = power(d2);
    s += e;
    u = __builtin_fmaf(e, fmaxf(d2, -1e30f), u);
  }
};

// Over the 64 lanes by moves inside the vector unit: rows of 16, the rows of a half,
// the halves; the last lane has it all. Six exchanges through LDS take as long as
// thirty of these.
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
__device__ __forceinline__ unsigned lanes_max(unsigned x) {
  return over_lanes((int)x, 0, [](int a, int b) {
    return (int)max((unsigned)a, (unsigned)b);
  });
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
  float u = f > 0.f ? f * __builtin_fmaf(a.s, d2, a.u) : 0.f;     // as raise
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

// A logit's log probability in a row of maximum m and sum of 2^logs: the difference is not
// scaled there and back, which would lose masked logits to -inf.
__device__ __forceinline__ float logprob(float x, float m, float logs) {
  return (x - m) - logs * LN2;
}

// What a row comes to. A token outside of the row has no log probability.
__device__ __forceinline__ void finish(const Sums& a, float xy, bool known,
                                       float* lp, float* ent, float* stat) {
  const float logs = __builtin_amdgcn_logf(a.s);       // log2
  *lp = known ? logprob(xy, a.m, logs) : __builtin_nanf("");
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
  auto one = [&](float v) {
    a.raise(v);
    a.add(v);
  };
  for (long long j = tid; j < head; j += CT) one(ds::to_f32(x[j]));
  long long j = tid;
  for (; j + (U - 1) * CT < nv; j += U * CT) {
    Chunk<T> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = stream(xv + j + i * CT);
    float t = LOWEST;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) t = fmaxf(t, ds::to_f32(v[i].v[e]));
    a.raise(t);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) a.add(ds::to_f32(v[i].v[e]));
  }
  for (; j < nv; j += CT) {
    const Chunk<T> v = xv[j];
#pragma unroll
    for (int e = 0; e < N; ++e) one(ds::to_f32(v.v[e]));
  }
  for (long long k = head + nv * N + tid; k < V; k += CT) one(ds::to_f32(x[k]));
  join_waves(a, lds);
  if (tid == 0) {
    const bool known = y >= 0 && y < V;
    finish(a, known ? ds::to_f32(x[y]) : 0.f, known, lp + row, ent + row,
           stat + 2 * row);
  }
}

// ------------------------------------------- few rows, or their best tokens too
//
// Parts of 8192 logits, held in registers: the sums of each, and its best, sorted.
// join_kernel makes a row of the parts.
//
// The best `top` of many, by lanes: the top-th largest of the lanes' own best is a
// bound that `top` logits reach, and what reaches it, few more than those, is
// gathered and put in its place by counting what is better. Taking one best after
// another cost 1.2 us each (24 x 128256 in all, us, 5 best 16.5 and now 15.2, 20 best 37
// and 20, 32 best 51 and 26); a single one is a maximum (128 rows 26.2 and 19.6).
// Bound by latency: the parts' kernel
// takes 4.7 us without best tokens, 10.5 with five, joining them 2.6 and 5.0.

// A logit and its id as one number: larger logits first, of equal ones the lower id.
// NaN lies above all, -0 is 0, and 0 stands for none.
typedef unsigned long long Rated;

__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);
  return x != x ? ~0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(Rated r) {
  const unsigned key = (unsigned)(r >> 32);
  return key == ~0u ? __builtin_nanf("")
                    : __builtin_bit_cast(
                          float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ Rated rated(unsigned key, int id) {
  return (Rated)key << 32 | (unsigned)~id;
}
__device__ __forceinline__ int id_of(Rated r) { return ~(int)(unsigned)r; }

__device__ __forceinline__ Rated of_lane(Rated x, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)x, lane);
  const unsigned hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
  return (Rated)hi << 32 | lo;
}
// How many of the first n lanes' are better, and the one that top - 1 are better than
// (1, which everything reaches, where there are fewer).
__device__ __forceinline__ int better(Rated x, int n) {
  int r = 0;
#pragma unroll 16
  for (int j = 0; j < n; ++j) r += of_lane(x, j) > x;
  return r;
}
__device__ __forceinline__ Rated bound(Rated x, int rank, int top) {
  const unsigned long long who = __ballot(rank == top - 1 && x != 0);
  return who ? of_lane(x, __builtin_ctzll(who)) : 1;
}
// Lanes that have one to add put it behind the n that are there; the new n.
__device__ __forceinline__ int gather(Rated* to, int n, Rated x, bool add) {
  const unsigned long long who = __ballot(add);
  if (add) {
    const int lane = threadIdx.x & 63;
    to[n + __builtin_popcountll(who & ((1ull << lane) - 1))] = x;
  }
  return n + __builtin_popcountll(who);
}
// Of n gathered ones of a wave, all different: each that fewer than `top` are better
// than, with their number.
template <typename F>
__device__ __forceinline__ void places(const Rated* from, int n, int top, F f) {
  for (int i = threadIdx.x & 63; i < n; i += 64) {
    const Rated x = from[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += from[j] > x;
    if (r < top) f(r, x);
  }
}

template <typename T>
__global__ __launch_bounds__(CT) void parts_kernel(
    const Rows rows, const long long* __restrict__ tokens,
    float* __restrict__ sums,          // [N, parts, 3]
    Rated* __restrict__ lists,         // [N, parts, top]
    const long long V, const int parts, const int top,
    const long long ignore) {
  constexpr int N = Chunk<T>::N, C = HELD / N, NW = CT / 64;
  extern __shared__ Rated room[];      // of each wave HELD top and top, then top
  __shared__ float lds[NW][3];
  const int row = blockIdx.x / parts, part = blockIdx.x % parts;
  const int tid = threadIdx.x;
  const int lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tokens[row] == ignore) return;
  const T* x = (const T*)rows.x + rows.at(row);
  // chunks lie on 16 bytes: the first and the last may reach out of the row
  const int ahead = (int)(((uintptr_t)x & 15) / sizeof(T));
  const long long first = (long long)part * PART + tid * N - ahead;
  float v[HELD];
  unsigned none = 0;                   // places that are none
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
        if (!in) none |= 1u << (c * N + e);
      }
    }
  }
  Sums a;
#pragma unroll
  for (int e = 0; e < HELD; ++e) a.m = fmaxf(a.m, v[e]);
#pragma unroll
  for (int e = 0; e < HELD; ++e) a.add(v[e]);
  join_waves(a, lds);
  if (tid == 0) {
    float* s = sums + ((long long)row * parts + part) * 3;
    s[0] = a.m;
    s[1] = a.s;
    s[2] = a.u;
  }
  if (top == 0) return;

  Rated* const held = room + wid * HELD * top;
  Rated* const best = room + NW * HELD * top;          // [waves][top]
  Rated* const all = best + NW * top;
  for (int i = tid; i < (NW + 1) * top; i += CT) best[i] = 0;
  // place e of the thread's is the logit first + at(e)
  auto at = [](int e) { return e / N * CT * N + e % N; };
  unsigned keys[HELD], key = 0;
  int place = 0;
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    keys[e] = none >> e & 1 ? 0u : key_of(v[e]);
    if (keys[e] > key) {
      key = keys[e];
      place = e;
    }
  }
  const Rated mine = key ? rated(key, (int)first + at(place)) : 0;
  if (top == 1) {
    const unsigned hi = lanes_max(key);
    const unsigned lo = lanes_max(key == hi ? (unsigned)mine : 0u);
    __syncthreads();
    if (lane == 0) best[wid] = (Rated)hi << 32 | lo;
  } else {
    const Rated low = bound(mine, better(mine, 64), top);
    const unsigned low_key = (unsigned)(low >> 32);
    int n = 0;
#pragma unroll
    for (int e = 0; e < HELD; ++e)
      if (__any(keys[e] >= low_key)) {
        const Rated r = rated(keys[e], (int)first + at(e));
        n = gather(held, n, r, keys[e] != 0 && r >= low);
      }
    __syncthreads();
    places(held, n, top, [&](int r, Rated y) { best[wid * top + r] = y; });
  }
  __syncthreads();
  // the waves' lists into one: a place in one's own, and in each of the others
  if (tid < NW * top && best[tid] != 0) {
    const Rated y = best[tid];
    int r = tid % top;
#pragma unroll
    for (int w = 0; w < NW; ++w)
      if (w != tid / top)
#pragma unroll 4
        for (int i = 0; i < top; ++i) r += best[w * top + i] > y;
    if (r < top) all[r] = y;
  }
  __syncthreads();
  if (tid < top) lists[((long long)row * parts + part) * top + tid] = all[tid];
}

// A wave a row; a lane a list, of the lists that there are in LDS.
__global__ __launch_bounds__(64) void join_kernel(
    const Rows rows, const int type, const long long* __restrict__ tokens,
    const float* __restrict__ sums, const Rated* __restrict__ lists,
    float* __restrict__ lp, float* __restrict__ ent, float* __restrict__ stat,
    float* __restrict__ top_lp, long long* __restrict__ top_ids,
    const long long V, const int parts, const int top,
    const long long ignore) {
  extern __shared__ Rated room[];      // [parts][top], then top (top + 1) / 2
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
  const Rated* from = lists + (long long)row * parts * top;
  for (int i = lane; i < parts * top; i += 64) room[i] = from[i];
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
  if (top == 0) return;
  __syncthreads();
  const Rated* const list = room + lane * top;
  // Where lists are few, the bound is one that deeper entries reach: deep + 1 of each of
  // the best half of the lists and more come to top.
  const int deep = min(top - 1, 2 * top / parts);
  const Rated down = lane < parts ? list[deep] : 0;
  const Rated low = bound(down, better(down, parts), (top + deep) / (deep + 1));
  const Rated head = lane < parts ? list[0] : 0;
  const int rank = better(head, parts);
  // an entry has its own list's earlier ones and better lists' heads before it
  Rated* const held = room + parts * top;
  int n = 0;
  for (int i = 0; i < top; ++i) {
    const bool may = lane < parts && rank + i < top;
    if (!__any(may)) break;
    const Rated e = may ? list[i] : 0;
    n = gather(held, n, e, e >= low);
  }
  __syncthreads();
  places(held, n, top, [&](int r, Rated e) {
    top_lp[out + r] = logprob(logit_of(e), a.m, logs);
    top_ids[out + r] = id_of(e);
  });
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
  if (glp && (y < 0 || y >= V)) g = __builtin_nanf("");
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
    Chunk<T> v = stream((const Chunk<T>*)(x + from + j * N));
#pragma unroll
    for (int e = 0; e < N; ++e)
      v.v[e] = one(ds::to_f32(v.v[e]), from + j * N + e);
    stream((Chunk<T>*)(d + from + j * N), v);
  }
  for (long long j = from + nv * N + tid; j < hi; j += CT)
    d[j] = one(ds::to_f32(x[j]), j);
}

}  // namespace

// Parts a row is cut into; 0: a workgroup a row, which saves a launch and the sums' way
// through memory. us, whole rows and parts, bf16: 16 x 32000 9.1 and 11.7, 384 x 32000
// 13.0 and 12.4, 16 x 128256 17.6 and 10.4, 128 26.3 and 15.5, 384 31.2 and 30.4,
// 512 32.0 and 37.9, 2048 85.7 and 134.5.
extern "C" int ds_logprobs_parts(int rows, long long V, int top) {
  const long long parts = (V + PART + 6) / PART;   // a row may begin inside a chunk
  return top == 0 && (parts <= 4 || rows >= 400) ? 0 : (int)parts;
}

// type: 0 fp32, 1 bf16, 2 fp16. parts as ds_logprobs_parts says, sums [N, parts, 3],
// lists [N, parts, top] of 8 bytes. Returns a hipError_t.
extern "C" int ds_logprobs_fwd(const void* x, long long outer_stride,
                               long long inner_stride, int inner, int type,
                               const long long* tokens, float* lp, float* ent,
                               float* stat, float* top_lp, long long* top_ids,
                               float* sums, void* lists, int rows, long long V,
                               int parts, int top, long long ignore,
                               void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Rows r = {x, outer_stride, inner_stride, inner};
  const int room = (CT / 64 * (HELD + 1) + 1) * top * (int)sizeof(Rated);
#define GO(T)                                                                  \
  if (parts == 0)                                                              \
    hipLaunchKernelGGL((rows_kernel<T>), dim3(rows), dim3(CT), 0, s, r,        \
                       tokens, lp, ent, stat, V, ignore);                      \
  else                                                                         \
    hipLaunchKernelGGL((parts_kernel<T>), dim3(parts * rows), dim3(CT), room,  \
                       s, r, tokens, sums, (Rated*)lists, V, parts, top, ignore)
  if (type == 0) { GO(float); }
  else if (type == 1) { GO(ds::bf16); }
  else { GO(ds::f16); }
#undef GO
  if (parts)
    hipLaunchKernelGGL(join_kernel, dim3(rows), dim3(64),
                       (parts * top + top * (top + 1) / 2) * sizeof(Rated), s,
                       r, type, tokens, sums, (const Rated*)lists, lp, ent,
                       stat, top_lp, top_ids, V, parts, top, ignore);
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
  // whole rows from 2048 on; fewer are cut, but not below 4096 logits. us, whole rows
  // and cut: 16 x 128256 33.3 and 8.4, 256 58.4 and 30.2, 1024 106.5 and 107.6; 256 x
  // 32000 18.3 and 10.8.
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
