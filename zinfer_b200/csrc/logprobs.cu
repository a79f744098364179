// Log probabilities of given tokens, with rank, entropy and the best alternatives, of rows of logits.
//
// With m = max x_j, S = sum e^(x_j - m) and T = sum e^(x_j - m) (x_j - m):
//   log p_t = (x_t - m) - ln S,   entropy = ln S - T / S,   rank_t = 1 + |{j : x_j before x_t}|,
// "before" being larger, or equal at a lower index.  S and T go from a maximum m to a larger m' by d = m - m':
// S' = e^d S, T' = e^d (T + d S); so ONE pass over a row gives all of them.  A row that holds NaN or +inf, or nothing above -inf,
// has no distribution: its numbers are NaN (what is not above -2^126 counts as -inf; where it holds NaN, its rank and alternatives
// mean nothing, an id of -1 among them).
//
// The best `top` of a row without sorting it and without a second pass: the pass also keeps, for each of some thousand groups of
// vectors (a thread's vectors in a quarter of its walk), the group's largest value and the first vector that has it.  The `top`-th
// largest of these pairs is a bound that `top` logits reach, so what is worse than it is not among the best, and what is
// not lies in the groups that reach the bound: only their vectors (1 in 50) are read again.  (First with the best pair of every
// thread, of which few are sorted, then, if too many groups reach that bound, with all of them.)  The few logits that pass are
// ranked by counting.  Exact whatever the values are: pairs are distinct, so equal logits cannot overrun the list.
//
// What bounds it: the logits' bytes once they are a few megabytes (a block per row, 16-byte loads, four under way per thread): 4,096
// rows of 65,536 float32 logits 159 us, 6.8 TB/s; of bfloat16, half the bytes, 105 us, the instructions of an exponential, two sums and
// the maxima per logit; with 20 alternatives 150.  Below that the chain of short steps: 64 float32 rows 6.7 us, with 20 alternatives
// 11; a row is then shared out over a cluster of up to eight blocks.
#include "common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

namespace {

constexpr int MOST_TOP = 32, MOST_VOCAB = 1 << 19, MOST_CLUSTER = 8;
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MOST_BLOCK = MOST_VOCAB / MOST_CLUSTER;       // logits a block walks
// a group holds at most 64 logits: a quarter of a walk of MOST_BLOCK logits, or a whole walk of a quarter of that.  The most
// that pass: those of the MOST_REACH groups that reach the bound and the at most 2 x 7 that no whole vector holds
constexpr int MOST_GROUP = MOST_BLOCK / THREADS / 4;
constexpr int MOST_REACH = 48, MOST_PASS = MOST_REACH * MOST_GROUP + 14;

typedef unsigned long long u64;

// Larger value first (-0 equals 0), NaN last.
__device__ __forceinline__ unsigned order_of(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);
  return v != v ? 0u : ((u & 0x80000000u) ? ~u : (u | 0x80000000u));
}
__device__ __forceinline__ float value_of(unsigned o) {
  return o == 0u ? NAN : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// (value, place): the lower place first among equal values
__device__ __forceinline__ u64 key_of(float v, unsigned place) { return ((u64)order_of(v) << 32) | (u64)(0xFFFFFFFFu - place); }
__device__ __forceinline__ unsigned place_of(u64 key) { return 0xFFFFFFFFu - (unsigned)key; }

// The larger of them, NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ unsigned max2_nan(unsigned a, unsigned b) {      // of two pairs of bfloat16
  unsigned r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float low_half(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(unsigned w) { return __uint_as_float(w & 0xffff0000u); }

// Stands for -inf, and for what lies below it, in the sums: -2^126, a number of both types.  Its weight is 0 like that of -inf, and 0
// times its difference from a maximum is 0 while that is finite: below 2^127.  From there on the numbers of both types lie 2^103 and more
// apart, so that whatever is less than the maximum weighs 0, and T, which 0 times an infinite difference may have made a NaN, is 0.
constexpr float LOWEST = -8.507059173023461586e37f, FAR = 1.7014118346046923173e38f;

// 16 bytes of logits, as they lie in memory until they are used.  `finite` gives the values as the sums take them, for bfloat16
// two with one maximum.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int E = 4;
  uint4 raw;
  __device__ __forceinline__ void values(float (&v)[4]) const {
    v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y), v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
  }
  __device__ __forceinline__ void finite(float (&v)[4]) const {
    values(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaxf(v[i], LOWEST);
  }
  __device__ __forceinline__ float most() const {
    return max_nan(max_nan(__uint_as_float(raw.x), __uint_as_float(raw.y)), __uint_as_float(raw.z), __uint_as_float(raw.w));
  }
};
template <> struct Vec<bf16> {
  static constexpr int E = 8;
  uint4 raw;
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = low_half(w[i]), v[2 * i + 1] = high_half(w[i]);
  }
  __device__ __forceinline__ void finite(float (&v)[8]) const {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned f = max2_nan(w[i], 0xfe80fe80u);
      v[2 * i] = low_half(f), v[2 * i + 1] = high_half(f);
    }
  }
  __device__ __forceinline__ float most() const {
    const unsigned m = max2_nan(max2_nan(raw.x, raw.y), max2_nan(raw.z, raw.w));
    return max_nan(low_half(m), high_half(m));
  }
};
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  return {__ldg(reinterpret_cast<const uint4*>(p))};
}

// e^d by one multiplication and ex2.approx: off by 2^-22 of it and the rounding of d log2(e)
__device__ __forceinline__ float exp_of(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
  return y;
}
// Pairs of float32, a product or sum of both in one instruction.
__device__ __forceinline__ u64 pair(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(u64 p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// A NaN among the logits is seen in m, which it makes NaN; +inf in m and in S.
struct Sums {
  float m;             // starts at LOWEST, and stays there where nothing is above it
  u64 S, T;            // two of each, for the logits at even and odd places
  __device__ __forceinline__ void move_to(float to) {
    to = max_nan(to, m);       // a NaN stays
    const float d = fmaxf(m - to, -1e4f), e = exp_of(d);       // 0 long before -1e4
    const u64 ee = pair(e, e);
    T = mul2(ee, fma2(pair(d, d), S, T));
    S = mul2(ee, S);
    m = to;
  }
  __device__ __forceinline__ void add(float x, float y) {      // neither of them -inf
    const u64 d = add2(pair(x, y), pair(-m, -m));
    const float2 l = halves(mul2(d, pair(1.4426950408889634f, 1.4426950408889634f)));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(l.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(l.y));
    const u64 ee = pair(e.x, e.y);
    S = add2(S, ee);
    T = fma2(ee, d, T);
  }
  __device__ __forceinline__ float sum() const { return halves(S).x + halves(S).y; }
  __device__ __forceinline__ float weighted() const { return halves(T).x + halves(T).y; }
};

// 32 keys, one to a lane, in order, the largest first.
__device__ __forceinline__ u64 swapped(u64 k, int with, bool keep_larger) {
  const u64 o = __shfl_xor_sync(0xffffffffu, k, with);
  return (k > o) == keep_larger ? k : o;
}
template <int N>
__device__ __forceinline__ void warp_sort(u64 (&k)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int with = size / 2; with; with /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) k[i] = swapped(k[i], with, ((lane & with) == 0) == ((lane & size) == 0 || size == 32));
}
// The 32 largest of two such lists, in order: the larger of a_i and b_(31 - i) are these, rising and falling.
__device__ __forceinline__ u64 warp_merge(u64 a, u64 b) {
  const int lane = threadIdx.x & 31;
  b = __shfl_xor_sync(0xffffffffu, b, 31);
  a = a > b ? a : b;
#pragma unroll
  for (int with = 16; with; with /= 2) a = swapped(a, with, (lane & with) == 0);
  return a;
}
// The 32 largest of the warps' lists, in the first warp; all threads call it, `s` holds a list per warp.
__device__ __forceinline__ u64 block_merge(u64 k, u64 (*s)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int w = WARPS / 2; w; w /= 2) {
    if (warp >= w && warp < 2 * w) s[warp][lane] = k;
    __syncthreads();
    if (warp < w) k = warp_merge(k, s[warp + w][lane]);
  }
  return k;
}

// What the blocks of a row's cluster tell the first one.
struct Told {
  float m, S, T;
  int before;
  u64 best[MOST_TOP];
};

// SEGS: the parts of a thread's walk that are groups of their own; 0: no alternatives are wanted.
template <typename T, int SEGS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 4)
    token_logprobs_kernel(const T* __restrict__ logits, long long ld, int V, const int* __restrict__ tokens,
                          float* __restrict__ logprob, int* __restrict__ rank, float* __restrict__ entropy, int top,
                          int* __restrict__ top_ids, float* __restrict__ top_logprobs, int* __restrict__ status) {
  constexpr int E = Vec<T>::E, U = 4, PARTS = SEGS ? SEGS : 1;
  constexpr bool TOP = SEGS > 0;
  __shared__ Told s_told;
  __shared__ float s_red[3][WARPS];
  __shared__ int s_before[WARPS];
  __shared__ u64 s_list[TOP ? WARPS : 1][32];
  __shared__ u64 s_pass[TOP ? MOST_PASS : 1];
  __shared__ int s_reach[MOST_REACH];
  __shared__ u64 s_bound;
  __shared__ int s_n_reach, s_n_pass;

  // Only a grid of some waves lets the next kernel start while it ends (4,096 rows 161 us a call, 166 without): the blocks of one that
  // starts beside a part of a wave lie unevenly over the SMs (331 rows, calls behind one another: 30 us, 18.6 without).
  if (gridDim.x >= 2048) zk_let_next_start();
  zk_wait_prior();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int parts = 1, part = 0;
  if (CLUSTER) {
    parts = (int)cg::this_cluster().num_blocks();
    part = (int)cg::this_cluster().block_rank();
  }
  const int row = blockIdx.x / parts;
  const T* x = logits + (size_t)row * ld;
  // logits [0, head) and [head + vecs * E, V) are single, those between are whole 16-byte vectors
  const int head = min(V, (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)));
  const int vecs = (V - head) / E;
  const int share = (vecs + parts - 1) / parts, v0 = min(vecs, part * share), v1 = min(vecs, v0 + share);
  const T* xv = x + head;
  const int tok = tokens[row];
  const bool known = tok >= 0 && tok < V;
  const float xt = known ? to_f32(x[tok]) : 0.f;
  const int tok_vec = tok < head ? -1 : (tok - head) / E;       // equal logits of vectors before it come before it

  // What comes before the token: above it, and in earlier vectors equal to it, that is above the number below it (for -inf
  // everything: nothing is at most NaN).
  const float late = xt, early = xt == -INFINITY ? NAN : nextafterf(xt, -INFINITY);
  Sums s{LOWEST, 0, 0};
  int before = 0;
  if (TOP && tid == 0) {
    s_bound = 0;
    s_n_reach = s_n_pass = 0;
  }
  // A thread's walk: vectors v0 + it * THREADS + tid, in batches of U of them, the next batch under way while one is worked on; whole
  // batches (all but the last) need no test per vector.  A group is a whole number of batches.
  const int its = (v1 - v0 + THREADS - 1) / THREADS, whole = (v1 - v0) / THREADS;
  const int per_seg = ((its + PARTS - 1) / PARTS + U - 1) / U * U;
  u64 group[PARTS];
  Vec<T> next[U];
  const T* ahead = xv + (size_t)(v0 + tid) * E;       // the batch to be requested
  auto request = [&](int it) {
    if (it + U <= whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = load_vec(ahead + u * (THREADS * E));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + (it + u) * THREADS + tid < v1) next[u] = load_vec(ahead + u * (THREADS * E));
    }
    ahead += U * THREADS * E;
  };
  request(0);
#pragma unroll
  for (int seg = 0; seg < PARTS; ++seg) {
    float g_max = NAN;
    int g_vec = -1;
    auto batch = [&](int it, int here) {      // `here` vectors, all where that is U
      const int first = v0 + it * THREADS + tid;
      Vec<T> f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = next[u];
      request(it + U);
      float mx[U], most = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mx[u] = u < here ? f[u].most() : -INFINITY;
        most = max_nan(most, mx[u]);
        if (TOP && u < here && (mx[u] > g_max || g_max != g_max)) {
          g_max = mx[u];
          g_vec = first + u * THREADS;
        }
      }
      if (!(most <= s.m)) s.move_to(most);
      if (!(most <= early)) {      // few vectors hold a logit that comes before the token
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float than = first + u * THREADS < tok_vec ? early : late;
          if (u >= here || mx[u] <= than) continue;
          float x[E];
          f[u].values(x);
#pragma unroll
          for (int e = 0; e < E; ++e) before += !(x[e] <= than);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= here) break;
        float x[E];
        f[u].finite(x);
#pragma unroll
        for (int e = 0; e < E; e += 2) s.add(x[e], x[e + 1]);
      }
    };
    int it = seg * per_seg;
    const int to = min(its, it + per_seg);
    for (; it + U <= min(to, whole); it += U) batch(it, U);
    if (it < to) {
      int here = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) here += v0 + (it + u) * THREADS + tid < v1;
      batch(it, here);
    }
    group[seg] = TOP && g_vec >= 0 ? key_of(g_max, g_vec) : 0ull;
  }
  // the single logits, and those equal ones in the token's own vector that come before it: the first block's
  if (part == 0) {
    const int single = V - vecs * E;
    if (tid < single) {
      const int j = tid < head ? tid : tid + vecs * E;
      const float v = to_f32(x[j]);
      if (!(v <= s.m)) s.move_to(v);
      s.add(fmaxf(v, LOWEST), LOWEST);
      if (s.m <= LOWEST) s.S = s.T = 0;      // (with m still LOWEST both weigh 1)
      before += v > xt || (v == xt && j < tok);
    }
    const int in_vec = tok - head - tok_vec * E;
    if (tid >= 32 && tid - 32 < in_vec && tok_vec >= 0 && tok_vec < vecs) before += to_f32(xv[(size_t)tok_vec * E + tid - 32]) == xt;
  }

  // the block's sums: everybody moves to the largest maximum
  float m = warp_max_nan(s.m);
  if (lane == 0) s_red[0][warp] = m;
  __syncthreads();
  m = warp_max_nan(lane < WARPS ? s_red[0][lane] : LOWEST);
  s.move_to(m);
  const float sum = warp_sum(s.sum()), weighted = warp_sum(s.weighted());
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) s_red[1][warp] = sum, s_red[2][warp] = weighted, s_before[warp] = before;

  if (TOP) {
    // The bound: the `top`-th of the threads' best groups (0: there are fewer), which more than `top` of all groups may reach, though
    // hardly ever many more; where they are, it is the `top`-th of all groups, which exactly `top` reach.
    auto bound_of = [&](u64 best) {
      best = block_merge(best, s_list);
      if (tid == top - 1) s_bound = best;
      if (tid == 0) s_n_reach = 0;
      __syncthreads();
      const u64 bound = s_bound;
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        if (group[i] && group[i] >= bound) {
          const int at = atomicAdd(&s_n_reach, 1);
          if (at < MOST_REACH) s_reach[at] = i * THREADS + tid;
        }
      __syncthreads();
      return bound;
    };
    u64 k[PARTS];
    k[0] = group[0];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) k[0] = k[0] > group[i] ? k[0] : group[i];
    u64 one[1] = {k[0]};
    warp_sort(one);
    u64 bound = bound_of(one[0]);
    if (PARTS > 1 && s_n_reach > MOST_REACH) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) k[i] = group[i];
      warp_sort(k);
#pragma unroll
      for (int i = 1; i < PARTS; ++i) k[0] = warp_merge(k[0], k[i]);
      __syncthreads();      // everybody has read the count
      bound = bound_of(k[0]);
    }
    const int again = s_n_reach * per_seg;
    for (int i = tid; i < again; i += THREADS) {
      const int grp = s_reach[i / per_seg], it = grp / THREADS * per_seg + i % per_seg;
      const int v = v0 + it * THREADS + grp % THREADS;
      if (it >= its || v >= v1) continue;
      float f[E];
      load_vec(xv + (size_t)v * E).values(f);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (key_of(f[e], v) >= bound) s_pass[atomicAdd(&s_n_pass, 1)] = key_of(f[e], head + v * E + e);
    }
    if (part == 0 && tid < V - vecs * E) {
      const int j = tid < head ? tid : tid + vecs * E;
      s_pass[atomicAdd(&s_n_pass, 1)] = key_of(to_f32(x[j]), j);
    }
    if (tid < top) s_told.best[tid] = 0;
    __syncthreads();
    const int n_pass = s_n_pass;
    for (int i = tid; i < n_pass; i += THREADS) {
      const u64 mine = s_pass[i];
      int ahead = 0;
      for (int j = 0; j < n_pass; ++j) ahead += s_pass[j] > mine;
      if (ahead < top) s_told.best[ahead] = mine;
    }
  }
  __syncthreads();
  if (tid == 0) {
    float S = 0.f, Tt = 0.f;
    int b = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) S += s_red[1][w], Tt += s_red[2][w], b += s_before[w];
    s_told.m = m;
    s_told.S = S;
    s_told.T = Tt;
    s_told.before = b;
  }
  if (CLUSTER) cg::this_cluster().sync();
  else __syncthreads();
  if (part == 0) {
    Sums all{LOWEST, 0, 0};
    int ahead = 0;
    if (lane < parts) {       // every warp: the sums are the same in all of them
      const Told* o = CLUSTER ? cg::this_cluster().map_shared_rank(&s_told, lane) : &s_told;
      all = {o->m, pair(o->S, 0.f), pair(o->T, 0.f)};
      ahead = o->before;
    }
    u64 best = 0;
    if (TOP) {                // warp w: block w's list
      if (warp < parts && lane < top) best = (CLUSTER ? cg::this_cluster().map_shared_rank(&s_told, warp) : &s_told)->best[lane];
      if (CLUSTER) best = block_merge(best, s_list);
    }
    if (warp == 0) {
      const float M = warp_max_nan(all.m);
      all.move_to(M);
      const float S = M > LOWEST ? warp_sum(all.sum()) : NAN, norm = logf(S);      // nothing above -inf: NaN
      const float weighted = warp_sum(all.weighted()), Tt = M >= FAR ? 0.f : weighted;
      ahead = __reduce_add_sync(0xffffffffu, ahead);
      if (lane == 0) {
        logprob[row] = known ? (xt - M) - norm : NAN;
        rank[row] = known ? 1 + ahead : 0;
        entropy[row] = norm - Tt / S;
        if (!known && status) atomicExch(status, 1);
      }
      if (TOP && lane < top) {
        top_ids[(size_t)row * top + lane] = (int)place_of(best);
        top_logprobs[(size_t)row * top + lane] = (value_of((unsigned)(best >> 32)) - M) - norm;
      }
    }
  }
  if (CLUSTER) cg::this_cluster().sync();      // the first block has read what the others told
}

template <typename T, int SEGS>
int launch(int parts, const T* logits, long long ld, int n, int V, const int* tokens, float* logprob, int* rank, float* entropy, int top,
           int* top_ids, float* top_logprobs, int* status, cudaStream_t stream) {
  if (parts == 1)
    return zk_launch_dependent(token_logprobs_kernel<T, SEGS, false>, dim3(n), dim3(THREADS), 0, stream, logits, ld, V, tokens,
                               logprob, rank, entropy, top, top_ids, top_logprobs, status);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * parts);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, SEGS, true>, logits, ld, V, tokens, logprob, rank, entropy, top,
                                 top_ids, top_logprobs, status);
}

template <typename T>
int launch_typed(const void* logits, long long ld, int n, int V, const int* tokens, float* logprob, int* rank, float* entropy, int top,
                 int* top_ids, float* top_logprobs, int* status, int sms, cudaStream_t stream) {
  // blocks per row: as many as give every SM two blocks, while a block has 2,048 logits and more; no block walks more than
  // MOST_BLOCK
  int parts = 1;
  while (parts < MOST_CLUSTER && ((long long)V > (long long)parts * MOST_BLOCK || ((long long)n * parts < 2 * sms && V / (2 * parts) >= 2048)))
    parts *= 2;
  if ((long long)n * parts > 0x7fffffffLL) return ZK_EINVAL;
  const T* x = (const T*)logits;
  if (top == 0) return launch<T, 0>(parts, x, ld, n, V, tokens, logprob, rank, entropy, top, top_ids, top_logprobs, status, stream);
  // a walk of at most MOST_GROUP logits per thread is one group, a longer one four
  const int vecs = V / Vec<T>::E, walk = ((vecs + parts - 1) / parts + THREADS - 1) / THREADS * Vec<T>::E;
  return walk <= MOST_GROUP ? launch<T, 1>(parts, x, ld, n, V, tokens, logprob, rank, entropy, top, top_ids, top_logprobs, status, stream)
                            : launch<T, 4>(parts, x, ld, n, V, tokens, logprob, rank, entropy, top, top_ids, top_logprobs, status, stream);
}

}  // namespace

extern "C" {

int zk_logprobs_most_top() { return MOST_TOP; }
int zk_logprobs_most_vocab() { return MOST_VOCAB; }

// logits [n, V], rows ld elements apart, dtype ZK_F32 or ZK_BF16; tokens [n].  An id outside [0, V) leaves NaN, rank 0 and
// status 1.  top_ids, top_logprobs [n, top].  sms: the device's SMs.
int zk_token_logprobs(const void* logits, long long ld, int n, int V, int dtype, const int* tokens, float* logprob, int* rank,
                      float* entropy, int top, int* top_ids, float* top_logprobs, int* status, int sms, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (V <= 0 || V > MOST_VOCAB || ld < 0 || top < 0 || top > MOST_TOP || top > V || !tokens || !logprob || !rank || !entropy ||
      (top > 0 && (!top_ids || !top_logprobs)) || (dtype != ZK_F32 && dtype != ZK_BF16) ||
      (uintptr_t)logits % (dtype == ZK_F32 ? 4 : 2))
    return ZK_EINVAL;
  return (dtype == ZK_F32 ? launch_typed<float> : launch_typed<bf16>)(logits, ld, n, V, tokens, logprob, rank, entropy, top, top_ids,
                                                                      top_logprobs, status, sms, stream);
}

}  // extern "C"
