// Attention of single-token steps whose sequences share prefixes over the paged cache.
//
// A group of sequences (answers to one prompt) holds the same first P positions in the same pages.  With
// scores s_j = cap(scale q . k_j), a row's softmax over its keys splits into the keys of the prefix and its own:
//   (m, l, o) of a set of keys = (max s_j, sum e^(s_j - m), sum e^(s_j - m) v_j),
//   of two sets: m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise; the result is o / l.
// So the prefix is walked once for the whole group, its rows being (sequence, head of the KV group) pairs, and every
// sequence's own keys on their own; both are cut into chunks that separate blocks walk, and `attn_shared_merge_kernel`
// joins what they leave (with the sink, one more term of l, and the gate).  The reference runs one sequence and has nothing
// of the kind; its single-token attention is cut and joined the same way (src/model.zig:1941-1955,
// src/attention.zig:749-814).
//
// The batch's sharing is described by `words` (int32, n rows): [0] the number of groups; from [4] on n / 2 records of four, a
// group's (first of its rows in the list below, number of rows, shared keys, first row), zeros behind the last group; then the list
// of the groups' rows, n entries; then for every row the first key that is its own (0: it shares nothing).  The kernels read it on the
// device, so that a recorded step serves every batch whose launch has the same shape.
#include "tcgen05.cuh"
#include <algorithm>
#include <atomic>
#include <math.h>

namespace {

struct SharedArgs {
  const void *q, *k, *v;
  void* out;
  float *part_o, *part_ml;          // [splits][n * H][vd], [splits][n * H][2] (maximum on base e, sum)
  const int *seq_start, *seq_slot, *page_table, *words;
  const float* sink;
  const void* gate;
  int* status;
  int pt_stride, n, H, Hkv, hd, vd, page_size, ld_gate;
  float scale, softcap;
  int chunk, n_tasks, shared_splits, own_splits, own_keys;   // n_tasks: blocks per KV head for the shared parts
  int G, page_shift;                // heads of a KV head; log2 of the page size, or -1
  int beside;                       // the kernel before this one is the groups' and nothing of it is read: see attn_shared_mma_kernel
};

__device__ __forceinline__ const int* rows_of(const SharedArgs& a) { return a.words + 4 + 4 * (a.n / 2); }
__device__ __forceinline__ int page_at(const SharedArgs& a, int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size; }
__device__ __forceinline__ const int* own_of(const SharedArgs& a) { return rows_of(a) + a.n; }

// What one block walks: rows [0, n_rows) of (sequence, head) pairs against keys [c0, c1) of one KV head.
struct Task {
  int kvh, split, c0, c1, n_rows, slot;      // slot: whose page table names the keys' pages
  const int* members;                        // the group's rows, or null: row `alone` only
  int first, alone;                          // the tile's first pair
};

// (What the batch says is read from L2: a kernel that starts beside the one before it meets no line that an SM kept.)
// Block -> task, a tile of `rows_per_tile` pairs of a group or `own_rows` of a sequence; the shared parts come first (they are
// the longest).  False: this block has nothing to do, with
// `t.split` >= 0 if its partials are to be marked empty.
__device__ __forceinline__ bool find_task(const SharedArgs& a, int rows_per_tile, int own_rows, Task& t) {
  const int G = a.G, n = a.n;
  const int n_shared = a.n_tasks * a.Hkv;
  if ((int)blockIdx.x < n_shared) {
    int i = blockIdx.x / a.Hkv;
    t.kvh = blockIdx.x % a.Hkv;
    const int lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < n / 2; g0 += 32) {       // 32 groups at a time: tasks of each, and their running sum
      const int4 rec = g0 + lane < n / 2 ? __ldcg(reinterpret_cast<const int4*>(a.words + 4) + g0 + lane) : make_int4(0, 0, 0, 0);
      const int cnt = (rec.y * G + rows_per_tile - 1) / rows_per_tile * ((rec.z + a.chunk - 1) / a.chunk);
      int upto = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto > i);
      if (past) {
        const int who = __ffs(past) - 1;
        const int local = i - __shfl_sync(0xffffffffu, upto - cnt, who);
        const int leader = __shfl_sync(0xffffffffu, rec.w, who);
        t.slot = __ldcg(a.seq_slot + leader);
        const int pairs = __shfl_sync(0xffffffffu, rec.y, who) * G;
        const int tiles = (pairs + rows_per_tile - 1) / rows_per_tile;
        const int c = local / tiles, tile = local % tiles;    // the tiles of a chunk beside one another: they read the same keys
        t.members = rows_of(a) + __shfl_sync(0xffffffffu, rec.x, who);
        t.first = tile * rows_per_tile;
        t.n_rows = min(rows_per_tile, pairs - t.first);
        t.split = c;
        t.c0 = c * a.chunk;
        t.c1 = min(__shfl_sync(0xffffffffu, rec.z, who), t.c0 + a.chunk);
        t.alone = -1;
        return true;
      }
      i -= __shfl_sync(0xffffffffu, upto, 31);
    }
    t.split = -1;
    return false;
  }
  // (few divisions: a block of two tiles of keys spends a fifth of its time here)
  unsigned i = blockIdx.x - n_shared, j = i / (unsigned)a.Hkv;
  t.kvh = (int)(i - j * a.Hkv);
  t.first = 0;
  if (G > own_rows) {      // a KV group of more heads than a tile has rows takes several tiles
    const unsigned tiles = (G + own_rows - 1) / own_rows;
    t.first = (int)(j % tiles) * own_rows;
    j /= tiles;
  }
  int b = (int)j, s = 0;
  if (a.own_splits > 1) {
    s = (int)(j / (unsigned)n);
    b = (int)j - s * n;
  }
  const int own = __ldcg(own_of(a) + b), L = __ldcg(a.seq_start + b) + 1;
  t.slot = __ldcg(a.seq_slot + b);
  if (s == 0 && t.kvh == 0 && t.first == 0 && L < own && threadIdx.x == 0 && a.status) atomicExch(a.status, 20);
  t.members = nullptr;
  t.alone = b;
  t.n_rows = min(own_rows, G - t.first);
  t.split = a.shared_splits + s;
  t.c0 = own;
  t.c1 = L;
  if (a.own_splits > 1) {
    t.c0 = own + s * a.own_keys;
    if (s + 1 < a.own_splits) t.c1 = min(L, t.c0 + a.own_keys);      // (the last one has what is left, however much was said to be)
  }
  return t.c1 > t.c0;
}

// The batch row and head of pair r of a task's tile.
__device__ __forceinline__ void pair_of(const SharedArgs& a, const Task& t, int r, int& b, int& head) {
  const int G = a.G, p = t.first + r;
  if (t.members) {
    const int m = (int)((unsigned)p / (unsigned)G);
    b = __ldcg(t.members + m);
    head = t.kvh * G + p - m * G;
  } else {
    b = t.alone;
    head = t.kvh * G + p;
  }
}

// A row without keys in its own chunk has the weight nothing there.
__device__ __forceinline__ void mark_empty(const SharedArgs& a, const Task& t) {
  if (t.split < 0) return;
  for (int r = threadIdx.x; r < t.n_rows; r += blockDim.x) {
    int b, head;
    pair_of(a, t, r, b, head);
    const size_t at = ((size_t)t.split * a.n + b) * a.H + head;
    a.part_ml[2 * at] = -INFINITY;
    a.part_ml[2 * at + 1] = 0.f;
  }
}

static long long blocks_of(const SharedArgs& a, int own_rows) {
  return (long long)a.Hkv * (a.n_tasks + (long long)a.n * ((a.G + own_rows - 1) / own_rows) * a.own_splits);
}

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // src-size 0: the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ------------------------------------------------------------------------------- any sizes, both types
// Float32 FMAs: a tile of R = 16 RT rows against 64 keys.  A thread holds RT rows x 4 keys of the scores (keys 16 apart, rows of
// K padded by 16 bytes), then RT rows x 4 values of every 64 of the result; threads without a row skip the arithmetic.  K and V
// lie in shared memory in their own type, two tiles of each: the next one is brought in by cp.async while this one is worked
// on, four threads to a row, so that no address needs a division (with loads that waited, a tile took some 5 us; 13 rows of
// 16 heads behind 900 to 2,500 keys, float32: 43 us a call then, 17 now).  Bound by reading K and V from shared memory, every warp all of a
// tile: 2.7 us of a tile's 6 are its scores' (at two blocks an SM).
constexpr int GK = 64, G_THREADS = 256;

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four(const bf16* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u));
}

// Row `row` (its thread's quarter `part`) of a tile from the cache; VEC: whole 16-byte pieces.
template <typename T, bool VEC>
__device__ __forceinline__ void bring_row(T* dst, const T* src, int width, int padded, bool there, int part) {
  if (VEC) {
    const int pieces = width * (int)sizeof(T) / 16;
    const unsigned d = smem_addr(dst);
    for (int i = part; i < pieces; i += 4) cp_async16(d + 16 * i, reinterpret_cast<const char*>(src) + 16 * i, there);
  } else {
    for (int i = part; i < padded; i += 4) dst[i] = there && i < width ? src[i] : from_f32<T>(0.f);
  }
}

template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(G_THREADS, 2) attn_shared_general_kernel(const SharedArgs a, int hdp, int vdp, int stages) {
  constexpr int R = 16 * RT, PAD = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char g_smem[];
  const int ldk = hdp + PAD, ldv = vdp + PAD;
  T* Ks = reinterpret_cast<T*>(g_smem);         // [stages][GK][ldk]
  T* Vs = Ks + stages * GK * ldk;               // [stages][GK][ldv]
  float* Qs = reinterpret_cast<float*>(Vs + stages * GK * ldv);      // [R][hdp]
  float* Ss = Qs + R * hdp;                     // [R][GK + 4]
  float* s_m = Ss + R * (GK + 4);               // [R] maximum, sum, factor
  float *s_l = s_m + R, *s_alpha = s_l + R;

  zk_wait_prior();
  Task t;
  const int tid = threadIdx.x;
  if (!find_task(a, R, R, t)) {
    mark_empty(a, t);
    return;
  }
  const T *q = (const T*)a.q, *kc = (const T*)a.k, *vc = (const T*)a.v;
  const int* pt = a.page_table + (size_t)t.slot * a.pt_stride;
  const int n_tiles = (t.c1 - t.c0 + GK - 1) / GK;
  const int row = tid >> 2;
  auto page_of = [&](int x) { return t.c0 + x * GK + row < t.c1 ? pt[page_at(a, t.c0 + x * GK + row)] : -1; };
  int next_page = page_of(0);      // of this thread's row of the tile that is brought next: on its way a tile ahead
  auto bring = [&](int x) {
    const int kp = t.c0 + x * GK + row, page = next_page;
    next_page = page_of(x + 1);
    if (kp < t.c1 && page < 0 && a.status) atomicExch(a.status, 2);
    const bool there = page >= 0;
    const size_t at = (((size_t)max(page, 0) * a.Hkv + t.kvh) * a.page_size + (there ? kp - page_at(a, kp) * a.page_size : 0));
    const int buf = stages == 2 ? x & 1 : 0;
    bring_row<T, VEC>(Ks + (buf * GK + row) * ldk, kc + at * a.hd, a.hd, hdp, there, tid & 3);
    bring_row<T, VEC>(Vs + (buf * GK + row) * ldv, vc + at * a.vd, a.vd, vdp, there, tid & 3);
    cp_async_commit();
  };
  bring(0);

  for (int r = tid >> 4; r < R; r += G_THREADS / 16) {
    int b = 0, head = 0;
    if (r < t.n_rows) pair_of(a, t, r, b, head);
    for (int d = tid & 15; d < hdp; d += 16)
      Qs[r * hdp + d] = r < t.n_rows && d < a.hd ? to_f32(q[((size_t)b * a.H + head) * a.hd + d]) * a.scale : 0.f;
  }
  for (int r = tid; r < R; r += G_THREADS) {
    s_m[r] = -INFINITY;
    s_l[r] = 0.f;
  }
  const int ty = tid >> 4, tx = tid & 15, warp = tid >> 5, lane = tid & 31;
  const bool mine = ty * RT < t.n_rows;
  float o[4][RT][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;

  for (int x = 0; x < n_tiles; ++x) {
    cp_async_wait<0>();
    __syncthreads();      // tile x has landed, and tile x - 1 is consumed
    if (stages == 2 && x + 1 < n_tiles) bring(x + 1);
    const int buf = stages == 2 ? x & 1 : 0;
    const T *Kt = Ks + buf * GK * ldk, *Vt = Vs + buf * GK * ldv;
    const int lim = t.c1 - (t.c0 + x * GK);      // keys of this tile
    if (mine) {
      float s[RT][4];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
      for (int d = 0; d < hdp; d += 4) {
        float4 qv[RT], kv[4];
#pragma unroll
        for (int i = 0; i < RT; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (ty * RT + i) * hdp + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) kv[j] = four(Kt + (tx + 16 * j) * ldk + d);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][j] = fmaf(qv[i].x, kv[j].x, fmaf(qv[i].y, kv[j].y, fmaf(qv[i].z, kv[j].z, fmaf(qv[i].w, kv[j].w, s[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = s[i][j];
          if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
          Ss[(ty * RT + i) * (GK + 4) + tx + 16 * j] = tx + 16 * j < lim ? v : -INFINITY;
        }
    }
    __syncthreads();
    for (int r = warp; r < t.n_rows; r += G_THREADS / 32) {
      float* row = Ss + r * (GK + 4);
      const float x0 = row[lane], x1 = row[lane + 32];
      const float m_old = s_m[r], m_new = fmaxf(m_old, warp_max(fmaxf(x0, x1)));
      const float p0 = x0 == -INFINITY ? 0.f : expf(x0 - m_new), p1 = x1 == -INFINITY ? 0.f : expf(x1 - m_new);
      row[lane] = p0;
      row[lane + 32] = p1;
      const float sum = warp_sum(p0 + p1);
      if (lane == 0) {
        const float al = m_new == -INFINITY ? 1.f : expf(m_old - m_new);
        s_alpha[r] = al;
        s_l[r] = s_l[r] * al + sum;
        s_m[r] = m_new;
      }
    }
    __syncthreads();
    if (mine) {
    float al[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) al[i] = ty * RT + i < t.n_rows ? s_alpha[ty * RT + i] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 4 * tx + 64 * j;
      if (d >= vdp) break;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][i][e] *= al[i];
#pragma unroll 2
      for (int k0 = 0; k0 < GK; k0 += 4) {
        float p[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const float4 pv = *reinterpret_cast<const float4*>(Ss + (ty * RT + i) * (GK + 4) + k0);
          p[i][0] = pv.x, p[i][1] = pv.y, p[i][2] = pv.z, p[i][3] = pv.w;
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const float4 vv = four(Vt + (k0 + kk) * ldv + d);
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            o[j][i][0] = fmaf(p[i][kk], vv.x, o[j][i][0]);
            o[j][i][1] = fmaf(p[i][kk], vv.y, o[j][i][1]);
            o[j][i][2] = fmaf(p[i][kk], vv.z, o[j][i][2]);
            o[j][i][3] = fmaf(p[i][kk], vv.w, o[j][i][3]);
          }
        }
      }
    }
    }
    if (stages == 1 && x + 1 < n_tiles) {
      __syncthreads();      // the only buffer is free
      bring(x + 1);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = ty * RT + i;
    if (r >= t.n_rows) continue;
    int b, head;
    pair_of(a, t, r, b, head);
    const size_t at = ((size_t)t.split * a.n + b) * a.H + head;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 4 * tx + 64 * j + e;
        if (d < a.vd) a.part_o[at * a.vd + d] = o[j][i][e];
      }
    if (tx == 0) {
      a.part_ml[2 * at] = s_m[r];
      a.part_ml[2 * at + 1] = s_l[r];
    }
  }
}

// ------------------------------------------------------------------------------- bfloat16, heads of 64 or 128: mma.sync
// Four warps walk the keys in tiles of 64 that lie inside one page, brought in by cp.async into a ring of XOR-swizzled
// buffers.  A block has 16 pairs, and every warp a quarter of a tile's keys for all of them; the warps' results meet at the
// end.  Keys outside the task's are zero-filled on load, so nothing stale reaches the arithmetic; only a task's first and last tile test the mask.  Softmax on base 2 with ex2.approx,
// maxima, sums and products in float32; the weights are rounded to bfloat16 (by 2^-8 of them at most) for P V.  Bound by the latency
// of a block's chain at few keys: 8 answers behind 960 tokens, 16 heads on 8, 3.4 us a block and 1.5 for the joining.
constexpr int TK = 64, M_WARPS = 4, M_THREADS = 32 * M_WARPS;

__device__ __forceinline__ void ldsm4(unsigned r[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(unsigned r[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma16816(float c[4], const unsigned a[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {      // 2^x on the special-function unit; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&t);
}
// Byte offset of 16-byte piece `ch` of row `r` in a tile of rows of HD bfloat16.
template <int HD>
__device__ __forceinline__ int swz(int r, int ch) {
  return r * (HD * 2) + ((ch & ~7) | ((ch ^ r) & 7)) * 16;
}

template <int HD>
constexpr int RING = HD == 64 ? 3 : 2;      // tile buffers

template <int HD>
__device__ __forceinline__ void walk_keys(const SharedArgs& a, const Task& t, unsigned char* smem) {
  constexpr int WK = M_WARPS, NST = RING<HD>;   // every warp has all rows and a quarter of a tile's keys
  constexpr int KW = TK / WK, NT = KW / 8;      // these, in groups of 8
  constexpr int KS = HD / 16, CH = HD / 8;
  constexpr int TILE = TK * HD * 2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const bf16 *q = (const bf16*)a.q, *kc = (const bf16*)a.k, *vc = (const bf16*)a.v;
  const int* pt = a.page_table + (size_t)t.slot * a.pt_stride;

  // Q fragments straight from global memory: rows g and g + 8
  unsigned qf[KS][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    int b = 0, head = 0;
    if (r < t.n_rows) pair_of(a, t, r, b, head);
    const bf16* src = q + ((size_t)b * a.H + head) * HD + 2 * c;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks][h] = r < t.n_rows ? __ldcg(reinterpret_cast<const unsigned*>(src + ks * 16)) : 0u;
      qf[ks][h + 2] = r < t.n_rows ? __ldcg(reinterpret_cast<const unsigned*>(src + ks * 16 + 8)) : 0u;
    }
  }

  // A thread's 16-byte pieces of a tile: piece n is row r0 + n * STEP, piece ch0 of it (STEP a multiple of 8: the swizzle
  // of all of them is the same)
  constexpr int PIECES = TK * CH / M_THREADS, STEP = M_THREADS / CH;
  static_assert(STEP % 8 == 0 && PIECES * STEP == TK, "pieces of a tile");
  const int r0 = tid / CH, ch0 = tid % CH;
  const unsigned sm_piece = smem_addr(smem) + swz<HD>(r0, ch0);
  const int g_piece = r0 * HD + ch0 * 8;

  const int k_begin = t.c0 / TK * TK, n_tiles = (t.c1 - k_begin + TK - 1) / TK;
  int ld_x = 0, ld_kb = k_begin, ld_in = k_begin - page_at(a, k_begin) * a.page_size;
  // the pages of 32 tiles at a time, a lane each, and those of the 32 behind them under way: asked for tile by tile, a number's way
  // from L2 was longer than a tile's work
  auto page_of = [&](int y) { return y < n_tiles ? __ldcg(pt + page_at(a, k_begin + y * TK)) : 0; };
  int pages = 0, next = page_of(lane);
  auto load_tile = [&](int buf) {
    if (ld_x % 32 == 0) {
      pages = next;
      next = page_of(ld_x + 32 + lane);
    }
    const int page = __shfl_sync(0xffffffffu, pages, ld_x % 32);
    if (page < 0 && tid == 0 && a.status) atomicExch(a.status, 2);
    const size_t base = (((size_t)(page < 0 ? 0 : page) * a.Hkv + t.kvh) * a.page_size + ld_in) * HD + g_piece;
    const bf16 *kg = kc + base, *vg = vc + base;
    const unsigned ks = sm_piece + buf * 2 * TILE, vs = ks + TILE;
    const bool whole = page >= 0 && ld_kb >= t.c0 && ld_kb + TK <= t.c1;
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
      const int kp = ld_kb + r0 + n * STEP;
      const bool valid = whole || (page >= 0 && kp >= t.c0 && kp < t.c1);
      cp_async16(ks + n * STEP * HD * 2, valid ? kg + n * STEP * HD : kc, valid);
      cp_async16(vs + n * STEP * HD * 2, valid ? vg + n * STEP * HD : vc, valid);
    }
    cp_async_commit();
    ++ld_x;
    ld_kb += TK;
    ld_in = ld_in + TK == a.page_size ? 0 : ld_in + TK;
  };

  const float scale2 = a.scale * 1.4426950408889634f;
  const float cap2 = a.softcap * 1.4426950408889634f, scale_cap = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, o[HD / 8][4];
#pragma unroll
  for (int j = 0; j < HD / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  for (int x = 0; x < NST - 1; ++x) {
    if (x < n_tiles) load_tile(x);
    else cp_async_commit();
  }
  for (int x = 0; x < n_tiles; ++x) {
    // every iteration commits one group: all but the newest NST - 2 have landed when tile x has
    cp_async_wait<NST - 2>();
    __syncthreads();       // tile x is there for all warps, and the buffer of tile x - 1 is free
    if (x + NST - 1 < n_tiles) load_tile((x + NST - 1) % NST);
    else cp_async_commit();
    const unsigned Kt = smem_addr(smem) + (x % NST) * 2 * TILE, Vt = Kt + TILE;
    const int kb = k_begin + x * TK;

    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks += 2) {
        unsigned f[4];
        ldsm4(f, Kt + swz<HD>(warp * KW + 8 * j + (lane & 7), 2 * ks + (lane >> 3)));
        mma16816(s[j], qf[ks], f[0], f[1]);
        mma16816(s[j], qf[ks + 1], f[2], f[3]);
      }
    }
    const bool edge = kb < t.c0 || kb + TK > t.c1;     // the same for the whole block
    float m_new[2] = {m_run[0], m_run[1]};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sc = s[j][e] * scale2;
        if (a.softcap > 0.f) sc = cap2 * fast_tanh(s[j][e] * scale_cap);
        if (edge) {
          const int kp = kb + warp * KW + 8 * j + 2 * c + (e & 1);
          if (kp < t.c0 || kp >= t.c1) sc = -INFINITY;
        }
        s[j][e] = sc;
        m_new[e >> 1] = fmaxf(m_new[e >> 1], sc);
      }
    float alpha[2], sub[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m_new[h] = fmaxf(m_new[h], __shfl_xor_sync(0xffffffffu, m_new[h], 1));
      m_new[h] = fmaxf(m_new[h], __shfl_xor_sync(0xffffffffu, m_new[h], 2));
      sub[h] = m_new[h] == -INFINITY ? 0.f : m_new[h];      // masked keys only so far: their weights stay 2^-inf = 0
      alpha[h] = ex2(m_run[h] - sub[h]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = ex2(s[j][e] - sub[e >> 1]);
        s[j][e] = p;
        sum[e >> 1] += p;
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l_run[h] = l_run[h] * alpha[h] + sum[h];      // this lane's share of the row; the quad adds up behind the loop
      m_run[h] = m_new[h];
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) {
        o[j][0] *= alpha[0];
        o[j][1] *= alpha[0];
        o[j][2] *= alpha[1];
        o[j][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      unsigned pa[4];
      pa[0] = pack_bf16(s[2 * kk][0], s[2 * kk][1]);
      pa[1] = pack_bf16(s[2 * kk][2], s[2 * kk][3]);
      pa[2] = pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]);
      pa[3] = pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
      for (int jn = 0; jn < HD / 8; jn += 2) {
        unsigned f[4];
        ldsm4_t(f, Vt + swz<HD>(warp * KW + 16 * kk + (lane & 7) + ((lane >> 3) & 1) * 8, jn + (lane >> 4)));
        mma16816(o[jn], pa, f[0], f[1]);
        mma16816(o[jn + 1], pa, f[2], f[3]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();       // the buffers are free: the warps that hold other keys of the same rows meet there
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  constexpr int LD = HD + 4;
  float* sm_o = reinterpret_cast<float*>(smem);            // [WK][16][LD]
  float2* sm_ml = reinterpret_cast<float2*>(sm_o + WK * 16 * LD);      // [WK][16]
  static_assert(WK * 16 * (LD * 4 + 8) <= 2 * NST * TILE, "the merge fits in the tile buffers");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + g + 8 * h;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j)
      *reinterpret_cast<float2*>(sm_o + r * LD + 8 * j + 2 * c) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
    if (c == 0) sm_ml[r] = make_float2(m_run[h], l_run[h]);
  }
  __syncthreads();
  for (int idx = tid; idx < t.n_rows * (HD / 4); idx += M_THREADS) {
    const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
    float2 ml[WK];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      ml[w] = sm_ml[w * 16 + r];
      M = fmaxf(M, ml[w].x);
    }
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float e = ml[w].x == -INFINITY ? 0.f : ex2(ml[w].x - M);
      const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * 16 + r) * LD + d);
      L = fmaf(e, ml[w].y, L);
      O.x = fmaf(e, v.x, O.x), O.y = fmaf(e, v.y, O.y), O.z = fmaf(e, v.z, O.z), O.w = fmaf(e, v.w, O.w);
    }
    int b, head;
    pair_of(a, t, r, b, head);
    const size_t at = ((size_t)t.split * a.n + b) * a.H + head;
    *reinterpret_cast<float4*>(a.part_o + at * HD + d) = O;
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(M * 0.6931471805599453f, L);
  }
}

// `beside`: the kernel before this one walks the groups' prefixes (tcgen05).  It lets this one start once all of its
// blocks have seen everything before them complete, so that both run side by side: this one reads only what those earlier
// kernels wrote, from L2, and writes what nobody else touches.  The kernel behind it waits for this one alone; so that this
// includes the groups' kernel, one block waits for that before it ends.
//
// Five blocks an SM for heads of 64: 96 registers, with which two find room beside a block of the groups' kernel (the compiler's own 121
// leave room for one: 64 answers behind 8,192 tokens 25.1 us, 23.7 so; six blocks 24.7).
template <int HD>
__global__ void __launch_bounds__(M_THREADS, HD == 64 ? 5 : 3) attn_shared_mma_kernel(const SharedArgs a) {
  extern __shared__ __align__(128) unsigned char mma_smem[];
  if (!a.beside) zk_wait_prior();
  Task t;
  if (find_task(a, 16, 16, t)) walk_keys<HD>(a, t, mma_smem);
  else mark_empty(a, t);
  if (a.beside && blockIdx.x == gridDim.x - 1) zk_wait_prior();
}

// Sets a kernel's shared-memory limit at its first launch on a device (a bit per device; a second thread sets the same).  `whole`: an SM
// gives its blocks all the shared memory it has, so that blocks of another kernel find room beside them.
template <typename K>
cudaError_t room_for(K kern, int smem, bool whole, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && whole) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ULL << dev, std::memory_order_relaxed);
  return e;
}

template <int HD>
int launch_mma(const SharedArgs& a, cudaStream_t stream) {
  constexpr int smem = RING<HD> * 2 * TK * HD * 2;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = room_for(attn_shared_mma_kernel<HD>, smem, true, done);
  if (e != cudaSuccess) return (int)e;
  const long long blocks = blocks_of(a, 16);
  if (blocks > 0x7fffffffLL) return ZK_EINVAL;
  return zk_launch_dependent(attn_shared_mma_kernel<HD>, dim3((unsigned)blocks), dim3(M_THREADS), smem, stream, a);
}

// ------------------------------------------------------------------------------- bfloat16 groups of many pairs: tcgen05
// Tiles of up to 128 pairs on the fifth-generation tensor cores, heads of 64 or 128.  Four warps serve: two bring K tiles of 64 keys, and
// V tiles, straight out of the pages with TMA (64 columns a box, 128-byte swizzle) into a ring of each, the page numbers 32 tiles at a
// time; an elected thread of the third issues S = Q K^T into the next of four score buffers in tensor memory, as far ahead as buffers
// are free; one of the fourth issues O += P V, with P as the A operand where its scores lay.  TWO groups of four softmax
// warps, a row per thread, take the even and the odd tiles, with a maximum, a sum and an O of their own, so that one
// group's exponentials run while the other loads, stores or waits; the two meet at the end like the chunks of different blocks do.
// O is rescaled, behind the exponentials, only in warps where a maximum has run 2^8 ahead; warps without a row of the tile only keep
// the barriers going.  Tiles of 64 or 32 pairs lie in the 128 rows two or four times: each of these PARTS weighs a half or a quarter of a
// tile's keys relative to a maximum of its own, and they are added up at the end, so that more warps share the exponentials: 6 groups of
// 9 answers, capped, 33.3 -> 28.9 us.  P V of a part's keys leaves the lanes of the other parts' rows alone: weights of 0 there would
// make a NaN of an infinite value.  The sequences' own keys are another kernel's,
// which runs beside this one: blocks that allocate no tensor memory, in one kernel with those that do, were held back until the others
// had ended.  Every wait on a barrier is bounded: a block that gives up records a code in *status, stops issuing, frees its tensor
// memory and returns.
//
// Bound by a softmax group's chain: 2,000 to 2,600 cycles for its tile, so half of that per tile, of which 512 are the exponentials' on
// the special-function unit (16 a cycle) and 128 (heads of 64) or 256 the products'; at many keys per SM then by DRAM: 12 groups of 6
// answers behind 16,384 tokens, 32 heads on 8 of 64, 73 us, 5.5 TB/s; heads of 128 behind 8,192, 78 us, 5.2 TB/s.  At few keys by a
// block's start and end, some 6 us: 64 answers behind 8,192 tokens 14.5 us, 13 of the 15 tiles in 8.  What was found on the way:
// one thread for both products and two score buffers: 65 -> 51 us (24 answers behind 32,768, heads of 128); a page number asked for
// tile by tile: 0.6 us of L2 in every tile's way; products issued under `lane == 0` 468 cycles a tile, under elect.sync 146;
// exponentials on the FMA units (every fourth: 1 to 6 % less, every second: more), the groups in turns: nothing gained.
using namespace tc5;

constexpr int T_ROWS = 128, T_SOFTMAX = 2 * T_ROWS, T_THREADS = T_SOFTMAX + 128;
constexpr int K_WARP = T_SOFTMAX / 32, V_WARP = K_WARP + 1, S_WARP = K_WARP + 2, PV_WARP = K_WARP + 3;
constexpr int BOX = TK * 128;                     // 64 keys x 64 columns
constexpr int NSB = 4;                            // score buffers
template <int HD>
struct T5 {
  static constexpr int ATOMS = HD / 64, Q_BYTES = T_ROWS * HD * 2, TILE = TK * HD * 2;
  static constexpr int NSTG = HD == 64 ? 6 : 3;   // tiles of K, and of V; leaves room on the SM for blocks of the kernel beside
  static constexpr int BARS = Q_BYTES + 2 * NSTG * TILE, ML = BARS + 512;
  static constexpr size_t SMEM = ML + 2 * T_ROWS * 8 + 1024 /*alignment*/;
  static constexpr unsigned S = 0, O = 64 * NSB, COLS = 512;      // tensor-memory columns: score buffers (P over them), two of O
  static_assert(O + 2 * HD <= COLS, "tensor memory");
};

__device__ __forceinline__ bool elect_one() {      // true in one lane of a whole warp
  unsigned p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Capped scores, cap * tanh(x) with x = score * scale / cap, as factors of the raw ones: where no x of the warp passes 0.4, which is
// what a cap is chosen for, tanh(x) = x (1 - u/3 + 2u^2/15 - 17u^3/315 + 62u^4/2835), u = x^2, off by 4e-7 at most (what fast_tanh is off
// by is 1e-6), in pairs of FMAs: the special-function unit, which bounds this kernel, would give three of its operations to
// every tanh.  Both leave score * scale, capped.
template <int N>
__device__ __forceinline__ void cap_scores(float (&sc)[N], float scale, float scale_cap, float cap, bool small) {
  if (small) {
    const float s2 = scale_cap * scale_cap, c1 = scale * (-1.f / 3.f) * s2, c2 = scale * (2.f / 15.f) * s2 * s2,
                c3 = scale * (-17.f / 315.f) * s2 * s2 * s2, c4 = scale * (62.f / 2835.f) * s2 * s2 * s2 * s2;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 s = make_float2(sc[j], sc[j + 1]), u = mul2(s, s);
      float2 y = fma2(make_float2(c4, c4), u, make_float2(c3, c3));
      y = fma2(y, u, make_float2(c2, c2));
      y = fma2(y, u, make_float2(c1, c1));
      y = mul2(s, fma2(y, u, make_float2(scale, scale)));
      sc[j] = y.x;
      sc[j + 1] = y.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) sc[j] = cap * fast_tanh(sc[j] * scale_cap);
  }
}

// 16 columns of this thread's lane; `tmem_put_wait` makes them seen.
__device__ __forceinline__ void tmem_put16(unsigned taddr, const float (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
               "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
               : "memory");
}
__device__ __forceinline__ void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_put8(unsigned taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

template <int HD, bool CAP, int PARTS>
__global__ void __maxnreg__(104)
    attn_shared_tc5_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedArgs a) {
  using L = T5<HD>;
  constexpr int PAIRS = T_ROWS / PARTS, NC = TK / PARTS;      // pairs of a tile; a tile's keys that a row weighs
  constexpr int NSTG = L::NSTG, TILE = L::TILE, ATOMS = L::ATOMS;
  extern __shared__ unsigned char t_smem[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)t_smem + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Task t;
  unsigned char *q_sm = base, *k_sm = base + L::Q_BYTES, *v_sm = k_sm + NSTG * TILE;
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(base + L::BARS);
  unsigned long long *q_full = bars, *k_full = bars + 1, *k_empty = k_full + NSTG, *v_full = k_empty + NSTG, *v_empty = v_full + NSTG,
                     *s_full = v_empty + NSTG, *p_ready = s_full + NSB, *pv_done = p_ready + NSB;
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(pv_done + NSB);
  static_assert(NSTG <= 6 && (1 + 4 * 6 + 3 * NSB) * 8 + 16 <= 512, "the barriers fit their bytes");
  volatile int* aborted = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (threadIdx.x == 0) {
    mbar_init(q_full, T_SOFTMAX);
    for (int s = 0; s < NSTG; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < NSB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], T_ROWS);
      mbar_init(&pv_done[i], 1);
    }
    *aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == S_WARP) tmem_alloc(tmem_slot, L::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_slot;
  zk_wait_prior();       // nothing of the kernels before is read, and nothing written, above this line
  zk_let_next_start();   // and only then may the next one start, which does not wait for them itself

  const bool work = find_task(a, PAIRS, 16, t);
  const int n_tiles = work ? (t.c1 - t.c0 + TK - 1) / TK : 0;      // c0 is a multiple of a tile
  // a wait of one of the four threads or of a softmax warp; false: given up (who waits for this one gives up after as long)
  auto wait = [&](unsigned long long* bar, int parity, int code) {
    if (mbar_wait(bar, parity & 1)) return true;
    atomicExch(a.status, code);
    *aborted = 1;
    return false;
  };
  // a whole warp's, which goes on or gives up as one
  auto warp_wait = [&](unsigned long long* bar, int parity, int code) { return __all_sync(0xffffffffu, wait(bar, parity, code)); };
  if (!work) {
  } else if (warp == K_WARP || warp == V_WARP) {
    const bool is_k = warp == K_WARP, lead = elect_one();
    const CUtensorMap* map = is_k ? &map_k : &map_v;
    unsigned char* to = is_k ? k_sm : v_sm;
    unsigned long long *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
    const int* pt = a.page_table + (size_t)t.slot * a.pt_stride;
    // the pages of 32 tiles at a time, a lane each, and those of the 32 behind them under way
    auto page_of = [&](int y) { return y < n_tiles ? __ldcg(pt + page_at(a, t.c0 + y * TK)) : 0; };
    int pages = 0, next = page_of(lane), x = 0;
    for (; x < n_tiles; ++x) {
      if (x % 32 == 0) {
        pages = next;
        next = page_of(x + 32 + lane);
      }
      const int s = x % NSTG, kb = t.c0 + x * TK;
      int page = __shfl_sync(0xffffffffu, pages, x % 32);
      if (page < 0) {               // a visible position without a page: the step's inputs are wrong, and so is its result
        if (lead) atomicExch(a.status, 2);
        page = 0;
      }
      const int row = (page * a.Hkv + t.kvh) * a.page_size + kb - page_at(a, kb) * a.page_size;
      if (!warp_wait(&empty[s], x / NSTG + 1, 14)) break;
      if (lead) {
        mbar_expect_tx(&full[s], TILE);
#pragma unroll
        for (int h = 0; h < ATOMS; ++h) tma_load_2d(to + s * TILE + h * BOX, map, 64 * h, row, &full[s]);
      }
    }
    if (x < n_tiles)                // given up: what was requested lands before the block ends
      for (int y = max(0, x - NSTG); y < x; ++y) mbar_wait(&full[y % NSTG], (y / NSTG) & 1);
  } else if (warp == S_WARP && elect_one()) {
    const unsigned idesc = instr_desc(T_ROWS, TK);                    // Q [128 x HD] . K^T: both K-major
    bool ok = wait(q_full, 0, 15);
    for (int x = 0; x < n_tiles && ok; ++x) {
      const int s = x % NSTG, sb = x % NSB;
      ok = wait(&k_full[s], x / NSTG, 15) && (x < NSB || wait(&pv_done[sb], x / NSB + 1, 13));      // P of tile x - 4 is read
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < ATOMS; ++h) {
        const unsigned long long dq = smem_desc(q_sm + h * (T_ROWS * 128)), dk = smem_desc(k_sm + s * TILE + h * BOX);
#pragma unroll
        for (int k = 0; k < 4; ++k)   // 32 bytes further along the swizzled rows per k step
          umma_bf16(tmem + L::S + 64u * (unsigned)sb, dq + (unsigned long long)(2 * k), dk + (unsigned long long)(2 * k), idesc,
                    h > 0 || k > 0 ? 1u : 0u);
      }
      umma_commit(&s_full[sb]);
      umma_commit(&k_empty[s]);
    }
  } else if (warp == PV_WARP && elect_one()) {
    const unsigned idesc = instr_desc(T_ROWS, 64) | (1u << 16);       // P [128 x 64 keys] . V: V is MN-major, 64 columns at a time
    for (int x = 0; x < n_tiles; ++x) {
      const int s = x % NSTG, sb = x % NSB;
      if (!wait(&v_full[s], x / NSTG, 15) || !wait(&p_ready[sb], x / NSB, 16)) break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < ATOMS; ++h) {
        const unsigned long long dv = smem_desc(v_sm + s * TILE + h * BOX);
#pragma unroll
        for (int k = 0; k < TK / 16; ++k) {   // P: 8 columns (16 keys) further; V: 16 key rows of 128 bytes further
          const unsigned to = tmem + L::O + (unsigned)(HD * (x & 1) + 64 * h), from = tmem + L::S + 64u * (unsigned)sb + 8u * (unsigned)k;
          if constexpr (PARTS == 1) {
            umma_bf16_ta(to, from, dv + (unsigned long long)(128 * k), idesc, (x > 1 || k > 0) ? 1u : 0u);
          } else {                            // these keys are one part's: only its rows' lanes take them
            unsigned off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) off[i] = 32 * i / PAIRS == 16 * k / NC ? 0u : ~0u;
            umma_bf16_ta_lanes(to, from, dv + (unsigned long long)(128 * k), idesc, (x > 1 || 16 * k % NC > 0) ? 1u : 0u, off);
          }
        }
      }
      umma_commit(&pv_done[sb]);
      umma_commit(&v_empty[s]);
    }
  } else if (warp < K_WARP) {
    const int r = threadIdx.x % T_ROWS, wg = threadIdx.x / T_ROWS;       // row of the tile = lane of tensor memory; even or odd tiles
    const int pair = r % PAIRS, part = r / PAIRS;      // (a warp is of one part)
    const bool row_ok = pair < t.n_rows, warp_ok = pair - lane < t.n_rows;
    int b = 0, head = 0;
    if (row_ok) pair_of(a, t, pair, b, head);
    {
      constexpr int HALF = HD / 16;      // 16-byte pieces of a row: each group brings one half
      const bf16* src = (const bf16*)a.q + ((size_t)b * a.H + head) * HD;
      const bool whole = (uintptr_t)a.q % 16 == 0;       // else on 4 bytes
#pragma unroll
      for (int i = 0; i < HALF; ++i) {
        const int ch = wg * HALF + i;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row_ok && whole) {
          v = reinterpret_cast<const uint4*>(src)[ch];
        } else if (row_ok) {
          const unsigned* w = reinterpret_cast<const unsigned*>(src) + 4 * ch;
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(q_sm + (ch / 8) * (T_ROWS * 128) + r * 128 + ((ch ^ r) & 7) * 16) = v;
      }
      fence_async_smem();
      mbar_arrive(q_full);
    }
    const unsigned lane_sel = (unsigned)(warp % 4 * 32) << 16;
    const unsigned tmem_o = tmem + L::O + (unsigned)(HD * wg) + lane_sel;
    // scores stay raw and the scale goes into the exponent, 2^((s - m) scale log2 e); capped ones are scaled as they are read
    const float c2 = (CAP ? 1.0f : a.scale) * 1.4426950408889634f;
    const float scale_cap = CAP ? a.scale / a.softcap : 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    // P V of tile x.  A barrier's parity tells its last phase only: the scores of tile x + 2 or x, seen before, show that the phase
    // before tile x's is complete (their buffers' P V four tiles back was waited for).
    auto pv_wait = [&](int x) {
      ok = warp_wait(&pv_done[x % NSB], x / NSB, 18);
      tc_fence_after();
      return ok;
    };
    for (int x = wg; x < n_tiles; x += 2) {
      const int kb = t.c0 + x * TK;
      const unsigned tmem_s = tmem + L::S + 64u * (unsigned)(x % NSB) + lane_sel;
      ok = warp_wait(&s_full[x % NSB], x / NSB, 17);
      if (!ok) break;
      tc_fence_after();
      if (warp_ok) {
        // (scores turn into weights in place and leave 16 columns at a time: 104 registers, with which two blocks of the kernel
        // beside find room on the SM, of heads of 128 one)
        float sc[NC];
        if constexpr (NC == 64) tmem_ld64(tmem_s, sc);
        else if constexpr (NC == 32) tmem_ld32(tmem_s + (unsigned)(32 * part), sc);
        else tmem_ld16(tmem_s + (unsigned)(16 * part), sc);
        const int lim = t.c1 - kb - part * NC;           // keys of these that the prefix has
        if (lim < NC) {
#pragma unroll
          for (int j = 0; j < NC; ++j) sc[j] = j < lim ? sc[j] : -INFINITY;
        }
        float m4[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
        for (int j = 4; j < NC; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) m4[e] = j + 4 + e < NC ? fmaxf(fmaxf(m4[e], sc[j + e]), sc[j + 4 + e]) : fmaxf(m4[e], sc[j + e]);
        float m_tile = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (CAP) {
          float a4[4] = {fabsf(sc[0]), fabsf(sc[1]), fabsf(sc[2]), fabsf(sc[3])};
#pragma unroll
          for (int j = 4; j < NC; j += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) a4[e] = fmaxf(a4[e], fabsf(sc[j + e]));
          // (masked keys make the tile that the prefix ends in one of large scores)
          const bool small = __all_sync(0xffffffffu, fmaxf(fmaxf(a4[0], a4[1]), fmaxf(a4[2], a4[3])) * scale_cap <= 0.4f);
          cap_scores(sc, a.scale, scale_cap, a.softcap, small);
          float m1[2] = {m_tile, m_tile};
          cap_scores(m1, a.scale, scale_cap, a.softcap, small);
          m_tile = m1[0];
          if (!small && lim < NC) {
#pragma unroll
            for (int j = 0; j < NC; ++j) sc[j] = j < lim ? sc[j] : -INFINITY;      // not -cap
            if (lim <= 0) m_tile = -INFINITY;
          }
        }
        // The maximum that weights are relative to follows the row's only where that is more than 2^8 ahead (weights stay below 256: as
        // many bits as ever): hardly a tile has a warp whose 32 rows all keep theirs otherwise.
        const bool move = (m_tile - m_run) * c2 > 8.0f;
        // both maxima scaled and rounded as the exponents below have them: what was summed relative to the old one is brought
        // to the new one exactly, however large the scores are
        const float mc_old = m_run == -INFINITY ? -INFINITY : m_run * c2;
        if (move) m_run = m_tile;
        const float mc = m_run == -INFINITY ? 0.f : m_run * c2;
        const float alpha = move ? ex2(mc_old - mc) : 1.0f;
        l_run *= alpha;
        const float2 c22 = make_float2(c2, c2), mc2 = make_float2(-mc, -mc);
        float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
        for (int h = 0; h < NC; h += 32) {
          constexpr int PIECE = NC < 32 ? NC : 32;
          float pk[PIECE / 2];      // pairs of bfloat16
#pragma unroll
          for (int j = h; j < h + PIECE; j += 4) {
            float2 u = fma2(make_float2(sc[j], sc[j + 1]), c22, mc2), v = fma2(make_float2(sc[j + 2], sc[j + 3]), c22, mc2);
            u.x = ex2(u.x);
            u.y = ex2(u.y);
            v.x = ex2(v.x);
            v.y = ex2(v.y);
            sum0 = add2(sum0, u);
            sum1 = add2(sum1, v);
            pk[(j - h) / 2] = __uint_as_float(pack_bf16(u.x, u.y));
            pk[(j - h) / 2 + 1] = __uint_as_float(pack_bf16(v.x, v.y));
          }
          // P lies where its scores lay; under the keys of other parts scores are left, which this row's lane never takes
          const unsigned to = tmem_s + (unsigned)(part * (NC / 2) + h / 2);
          if constexpr (PIECE == 32) tmem_put16(to, pk);
          else tmem_put8(to, pk);
        }
        l_run += (sum0.x + sum0.y) + (sum1.x + sum1.y);
        tmem_put_wait();
        if (x >= 2 && __any_sync(0xffffffffu, move)) {    // O follows the new maximum once P V of this group's tile before is complete
          if (!pv_wait(x - 2)) break;
#pragma unroll
          for (int c0 = 0; c0 < HD; c0 += 32) {
            float o[32];
            tmem_ld32(tmem_o + (unsigned)c0, o);
            unsigned w[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(o[j] * alpha);
            tmem_st32(tmem_o + (unsigned)c0, w);
          }
        }
      }
      if (kb + TK > t.c1) {        // what lies behind the prefix weighs 0, but 0 times a stale NaN would not be
        const int first = t.c1 - kb;
        ok = warp_wait(&v_full[x % NSTG], x / NSTG, 15);      // V has landed
        if (!ok) break;
        for (int i = r; i < (TK - first) * 8 * ATOMS; i += T_ROWS)
          *reinterpret_cast<uint4*>(v_sm + x % NSTG * TILE + (i % ATOMS) * BOX + (first + i / ATOMS / 8) * 128 + (i / ATOMS % 8) * 16) =
              make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      tc_fence_before();
      mbar_arrive(&p_ready[x % NSB]);
    }
    // The two groups' results of a row: maximum and sum through shared memory; O lies in tensor memory for both to read, once the
    // last P V of each is seen complete by its own group.
    if (ok && warp_ok && n_tiles > wg) pv_wait((n_tiles - 1 - wg) / 2 * 2 + wg);
    float2* ml = reinterpret_cast<float2*>(base + L::ML);
    ml[wg * T_ROWS + r] = make_float2(m_run == -INFINITY ? -INFINITY : m_run * c2, l_run);
    tc_fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(T_SOFTMAX) : "memory");
    tc_fence_after();
    ok = ok && !*aborted;
    ok = __all_sync(0xffffffffu, ok);
    // through shared memory (the tiles are all consumed): a row's values leave side by side.  Stored from the lanes' rows, every
    // instruction met 32 lines, and a block took 2.1 us for it.
    constexpr int HALF = HD / 2, LD = HALF + 4, LANES = HALF / 4;      // each group joins and stores one half of the columns
    float* stage = reinterpret_cast<float*>(k_sm) + wg * T_ROWS * LD;
    long long* places = reinterpret_cast<long long*>(q_sm);
    static_assert(2 * T_ROWS * LD * 4 <= 2 * NSTG * TILE, "the rows fit where the tiles lay");
    if (ok && warp_ok) {   // uniform in the warp
      float M = -INFINITY, sum = 0.f;
#pragma unroll
      for (int q = 0; q < 2 * PARTS; ++q) M = fmaxf(M, ml[q * PAIRS + pair].x);      // (the second group's behind the first's)
      float f[2] = {0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 2 * PARTS; ++q) {
        const float2 v = ml[q * PAIRS + pair];
        const float e = v.x == -INFINITY ? 0.f : ex2(v.x - M);
        sum = fmaf(e, v.y, sum);
        if (q % PARTS == part) f[q / PARTS] = e;
      }
      if (row_ok && wg == 0 && part == 0) {
        const long long at = ((long long)t.split * a.n + b) * a.H + head;
        places[pair] = at;
        *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(M * 0.6931471805599453f, sum);
      }
#pragma unroll
      for (int c0 = 0; c0 < HALF; c0 += 16) {
        float o[16];
        tmem_ld16(tmem + L::O + lane_sel + (unsigned)(wg * HALF + c0), o);
        if (n_tiles > 1) {
          float o1[16];
          tmem_ld16(tmem + L::O + (unsigned)HD + lane_sel + (unsigned)(wg * HALF + c0), o1);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = fmaf(f[0], o[i], f[1] * o1[i]);
        } else if (PARTS > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= f[0];
        }
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(stage + r * LD + c0 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
    }
    unsigned all_ok;       // places and rows are read across warps: all of them, or nothing
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.and.pred q, 1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(all_ok)
                 : "r"(ok ? 1u : 0u), "n"(T_SOFTMAX)
                 : "memory");
    if (all_ok)
      for (int i = r; i < t.n_rows * LANES; i += T_ROWS) {
        const int p = i / LANES, c = i % LANES * 4;
        float4 v = *reinterpret_cast<const float4*>(stage + p * LD + c);
#pragma unroll
        for (int q = 1; q < PARTS; ++q) {
          const float4 w = *reinterpret_cast<const float4*>(stage + (q * PAIRS + p) * LD + c);
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        *reinterpret_cast<float4*>(a.part_o + places[p] * HD + wg * HALF + c) = v;
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == S_WARP) tmem_dealloc(tmem, L::COLS);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

template <int HD, int PARTS>
int launch_tc5(const SharedArgs& a, long long num_pages, cudaStream_t stream) {
  if (a.n_tasks == 0) return launch_mma<HD>(a, stream);      // nothing is shared
  EncodeTiledFn fn = encode_fn();
  const long long blocks = (long long)a.n_tasks * a.Hkv;
  if (!fn || blocks > 0x7fffffffLL || !a.status || num_pages <= 0 || a.chunk % TK) return ZK_EINVAL;
  CUtensorMap map[2];
  for (int which = 0; which < 2; ++which) {
    const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)num_pages * a.Hkv * a.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)TK}, estr[2] = {1, 1};
    if (dims[1] > 0x7fffffffULL ||
        fn(&map[which], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(which ? a.v : a.k), dims, strides, box, estr,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return ZK_EINVAL;
  }
  static std::atomic<unsigned long long> done[2];
  const bool cap = a.softcap > 0.f;
  auto kern = cap ? attn_shared_tc5_kernel<HD, true, PARTS> : attn_shared_tc5_kernel<HD, false, PARTS>;
  const cudaError_t e = room_for(kern, (int)T5<HD>::SMEM, true, done[cap]);
  if (e != cudaSuccess) return (int)e;
  const int rc = zk_launch_dependent(kern, dim3((unsigned)blocks), dim3(T_THREADS), T5<HD>::SMEM, stream, map[0], map[1], a);
  if (rc) return rc;
  SharedArgs own = a;
  own.n_tasks = 0;
  own.beside = 1;
  return launch_mma<HD>(own, stream);
}

// ------------------------------------------------------------------------------- joining the partial results
// A warp per (row, head).  A row of a group has partials in the splits [0, ceil(own / chunk)), own being the keys it
// shares, and every row in the own splits behind `shared_splits`; they are added in that order.
template <typename T>
__global__ void attn_shared_merge_kernel(const SharedArgs a) {
  zk_let_next_start();
  zk_wait_prior();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int n_rows = a.n * a.H;
  if (row >= n_rows) return;
  const int b = row / a.H, head = row % a.H;
  const int mine = (own_of(a)[b] + a.chunk - 1) / a.chunk;     // the splits its group's prefix has
  const int count = mine + a.own_splits;
  auto at = [&](int i) { return (size_t)(i < mine ? i : a.shared_splits + i - mine) * n_rows + row; };
  float M = a.sink ? a.sink[head] : -INFINITY;
  for (int i = lane; i < count; i += 32) M = fmaxf(M, a.part_ml[2 * at(i)]);
  M = warp_max(M);
  float L = a.sink && a.sink[head] != -INFINITY ? expf(a.sink[head] - M) : 0.f, acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  for (int i0 = 0; i0 < count; i0 += 32) {
    float e = 0.f, le = 0.f;      // lane i: split i0 + i
    if (i0 + lane < count) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at(i0 + lane));
      e = ml.x == -INFINITY ? 0.f : expf(ml.x - M);
      le = e * ml.y;
    }
    L += warp_sum(le);
    const int here = min(32, count - i0);
    for (int u0 = 0; u0 < here; u0 += 4) {      // four splits' rows under way
      float w[4], v[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        w[u] = u0 + u < here ? __shfl_sync(0xffffffffu, e, (u0 + u) & 31) : 0.f;
        const float* po = a.part_o + at(i0 + u0 + u) * a.vd;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u][j] = w[u] != 0.f && lane + 32 * j < a.vd ? po[lane + 32 * j] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = fmaf(w[u], v[u][j], acc[j]);
    }
  }
  float inv = L == 0.f ? 0.f : 1.0f / L;      // (a NaN stays one)
  if (a.gate) inv /= 1.0f + expf(-to_f32(((const T*)a.gate)[(size_t)b * a.ld_gate + head]));
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (lane + 32 * j < a.vd) ((T*)a.out)[(size_t)row * a.vd + lane + 32 * j] = from_f32<T>(acc[j] * inv);
}

// The same for values 64 and 128 wide: four values to a lane, HD / 4 lanes and four such sets of lanes to a row; set s takes the
// splits s, s + 4, ..., up to four of them under way at a time, and the sets meet in shared memory, in their order (208 rows of 20
// to 40 splits, float32: 3.3 us sooner done than by the kernel above).  Who shares how much was written before the kernel in front of this one
// began, which waited for it: it is read while that one ends.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attn_shared_merge_rows_kernel(const SharedArgs a) {
  constexpr int LANES = HD / 4, SETS = 4, ROWS = 128 / (LANES * SETS), U = 4;
  __shared__ float4 s_acc[ROWS][SETS][LANES];
  __shared__ float2 s_ml[ROWS][SETS];
  zk_let_next_start();
  const int lane = threadIdx.x % LANES, set = threadIdx.x / LANES % SETS, r = threadIdx.x / (LANES * SETS);
  const int n_rows = a.n * a.H, row = min(n_rows - 1, (int)blockIdx.x * ROWS + r);
  const int b = row / a.H, head = row % a.H;
  const int mine = (__ldcg(own_of(a) + b) + a.chunk - 1) / a.chunk, count = mine + a.own_splits;
  zk_wait_prior();
  auto at = [&](int i) { return (size_t)(i < mine ? i : a.shared_splits + i - mine) * n_rows + row; };
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = set; i0 < count; i0 += SETS * U) {
    float2 ml[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + SETS * u < count) {
        const size_t p = at(i0 + SETS * u);
        ml[u] = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
        v[u] = *reinterpret_cast<const float4*>(a.part_o + p * HD + 4 * lane);
      }
    }
    float m = M;
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(m, ml[u].x);
    const float f = M == -INFINITY ? 0.f : expf(M - m);
    L *= f;
    acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
    M = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].y == 0.f) continue;       // an empty chunk's row was not written
      const float e = expf(ml[u].x - m);
      L = fmaf(e, ml[u].y, L);
      acc.x = fmaf(e, v[u].x, acc.x), acc.y = fmaf(e, v[u].y, acc.y), acc.z = fmaf(e, v[u].z, acc.z), acc.w = fmaf(e, v[u].w, acc.w);
    }
  }
  s_acc[r][set][lane] = acc;
  if (lane == 0) s_ml[r][set] = make_float2(M, L);
  __syncthreads();
  if (set > 0 || (int)blockIdx.x * ROWS + r >= n_rows) return;
  M = a.sink ? a.sink[head] : -INFINITY;
#pragma unroll
  for (int s = 0; s < SETS; ++s) M = fmaxf(M, s_ml[r][s].x);
  L = a.sink && a.sink[head] != -INFINITY ? expf(a.sink[head] - M) : 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    const float e = s_ml[r][s].x == -INFINITY ? 0.f : expf(s_ml[r][s].x - M);
    const float4 v = s_acc[r][s][lane];
    L = fmaf(e, s_ml[r][s].y, L);
    acc.x = fmaf(e, v.x, acc.x), acc.y = fmaf(e, v.y, acc.y), acc.z = fmaf(e, v.z, acc.z), acc.w = fmaf(e, v.w, acc.w);
  }
  float inv = L == 0.f ? 0.f : 1.0f / L;      // (a NaN stays one)
  if (a.gate) inv /= 1.0f + expf(-to_f32(((const T*)a.gate)[(size_t)b * a.ld_gate + head]));
  T* to = (T*)a.out + (size_t)row * HD + 4 * lane;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  else
    *reinterpret_cast<float4*>(to) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <typename T, int RT, bool VEC>
int launch_general_as(const SharedArgs& a, cudaStream_t stream) {
  const int hdp = (a.hd + 3) / 4 * 4, vdp = (a.vd + 3) / 4 * 4, R = 16 * RT, pad = 16 / (int)sizeof(T);
  auto bytes = [&](int h, int v, int stages) { return stages * GK * (h + v + 2 * pad) * sizeof(T) + (size_t)(R * h + R * (GK + 4) + 3 * R) * 4; };
  auto kern = attn_shared_general_kernel<T, RT, VEC>;
  static std::atomic<unsigned long long> done{0};
  const int most = (int)std::min<size_t>(bytes(256, 256, 2), 227 * 1024), stages = bytes(hdp, vdp, 2) <= (size_t)most ? 2 : 1;
  const cudaError_t e = room_for(kern, most, false, done);
  if (e != cudaSuccess) return (int)e;
  const long long blocks = blocks_of(a, R);
  if (blocks > 0x7fffffffLL) return ZK_EINVAL;
  return zk_launch_dependent(kern, dim3((unsigned)blocks), dim3(G_THREADS), bytes(hdp, vdp, stages), stream, a, hdp, vdp, stages);
}
template <typename T>
int launch_general(const SharedArgs& a, int tile_rows, cudaStream_t stream) {
  const bool vec = a.hd * sizeof(T) % 16 == 0 && a.vd * sizeof(T) % 16 == 0 && (uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0;
  if (tile_rows == 16) return vec ? launch_general_as<T, 1, true>(a, stream) : launch_general_as<T, 1, false>(a, stream);
  return vec ? launch_general_as<T, 2, true>(a, stream) : launch_general_as<T, 2, false>(a, stream);
}

// What the tensor cores take: the sizes for which single-token attention without shared prefixes rounds its weights to bfloat16 too.
// More than 16 heads to a KV head run on float32 FMAs there, and so they do here: a fork's steps are as exact as a sequence's own.
static bool mma_takes(int dtype, int G, int hd, int vd, int page_size) {
  return dtype == ZK_BF16 && G <= 16 && hd == vd && (hd == 64 || hd == 128) && page_size % TK == 0;
}

template <int HD>
int launch_rows(const SharedArgs& a, int tile_rows, long long num_pages, cudaStream_t stream) {
  switch (tile_rows) {
    case 16: return launch_mma<HD>(a, stream);
    case 32:
      if constexpr (HD == 64) return launch_tc5<HD, 4>(a, num_pages, stream);
      return ZK_EINVAL;
    case 64: return launch_tc5<HD, 2>(a, num_pages, stream);
    case 128: return launch_tc5<HD, 1>(a, num_pages, stream);
    default: return ZK_EINVAL;
  }
}

template <typename T>
int launch_merge(const SharedArgs& a, cudaStream_t stream) {
  const int warps = 4;
  if ((a.vd == 64 || a.vd == 128) && (uintptr_t)a.out % (4 * sizeof(T)) == 0)
    return zk_launch_dependent(a.vd == 64 ? attn_shared_merge_rows_kernel<T, 64> : attn_shared_merge_rows_kernel<T, 128>,
                               dim3(a.vd == 64 ? ceil_div_i(a.n * a.H, 2) : a.n * a.H), dim3(128), 0, stream, a);
  return zk_launch_dependent(attn_shared_merge_kernel<T>, dim3(ceil_div_i(a.n * a.H, warps)), dim3(warps * 32), 0, stream, a);
}

}  // namespace

extern "C" {

// (sequence, head) pairs that one block's tile of a group holds; `pairs`: the most pairs a group has, `longest`: the keys of the longest
// prefix.  Tiles of 32, 64 and 128 are the tcgen05 kernel's, tiles of 16 the mma.sync one's (both: bfloat16 heads of 64 or 128, at most 16
// to a KV head, and pages of whole key tiles).  A tile of 16 costs less to start, so it serves groups that fit one, unless their keys are
// many, and few keys of two (8 KV heads, one group, us): heads of 64, tiles of 16 / 32: 8 pairs behind 1,024 keys 5.9 / 7.5, behind 4,096
// 9.5 / 8.9, 16 pairs 6.9 / 7.8, 11.2 / 9.1, 32 behind 256 7.7 / 7.8, behind 1,024 9.1 / 8.3; heads of 128, tiles of 16 / 64: 8 pairs 7.3
// / 8.4, 12.0 / 10.1, 16 behind 256 9.3 / 8.2.  Smaller tcgen05 tiles share a row's keys out over more warps: six groups of 32 pairs
// behind 16,384 keys, tiles of 32 / 64 / 128: heads of 64 40 / 40 / 52, behind 4,096 16.4 / 17.2 / 20.9, of 128 25.9 / 25.4 / 26.5 there.
// Other types and heads: 32 rows a block on FMAs, 16 where that holds all.
int zk_attn_shared_tile_rows(int dtype, int G, int hd, int vd, int page_size, int pairs, int longest) {
  if (!mma_takes(dtype, G, hd, vd, page_size)) return pairs > 16 ? 32 : 16;
  const bool tc5 = hd == 128 ? pairs > 8 || longest >= 4096
                             : longest >= (pairs > 16 ? 1024 : pairs > 8 ? 2048 : 4096) || pairs > 32;
  return !tc5 ? 16 : pairs > 64 ? 128 : pairs > 32 || hd == 128 ? 64 : 32;
}

// q, out [n, H * hd] and [n, H * vd]; k, v the paged cache of num_pages pages; `words` as described above, on 16 bytes.  `sizes` (host
// memory): n, H, Hkv, hd, vd, page_size, pt_stride, ld_gate, chunk, n_tasks, shared_splits, own_splits, own_keys, tile_rows, dtype.
// chunk: keys of a prefix per block; n_tasks: at least the tiles times chunks of all groups; shared_splits: at least the chunks of
// the longest prefix.  A row's own keys are cut every own_keys keys from its first own one, own_splits chunks that must reach the
// longest row's last key.  part_o (on 16 bytes) and part_ml: (shared_splits + own_splits) * n * H rows.  `status` gets 20 where
// a row is shorter than the prefix it shares, 2 where a key has no page.  tile_rows: what zk_attn_shared_tile_rows said.
int zk_attn_shared(const void* q, const void* k, const void* v, void* out, float* part_o, float* part_ml, const int* seq_start,
                   const int* seq_slot, const int* page_table, const int* words, const float* sink, const void* gate, int* status,
                   const int* sizes, float scale, float softcap, long long num_pages, cudaStream_t stream) {
  if (!sizes) return ZK_EINVAL;
  const int n = sizes[0], H = sizes[1], Hkv = sizes[2], hd = sizes[3], vd = sizes[4], page_size = sizes[5], pt_stride = sizes[6],
            ld_gate = sizes[7], chunk = sizes[8], n_tasks = sizes[9], shared_splits = sizes[10], own_splits = sizes[11],
            own_keys = sizes[12], tile_rows = sizes[13], dtype = sizes[14];
  if (n <= 0) return 0;
  if (H <= 0 || Hkv <= 0 || H % Hkv || hd <= 0 || vd <= 0 || hd > 256 || vd > 256 || page_size <= 0 || !words || !part_o ||
      !part_ml || chunk <= 0 || n_tasks < 0 || shared_splits < 0 || own_splits < 1 || (own_splits > 1 && own_keys <= 0) ||
      (n_tasks > 0 && shared_splits < 1) || (uintptr_t)part_o % 16 || (uintptr_t)part_ml % 8 || (uintptr_t)words % 16 ||
      (gate && ld_gate < H) || (long long)n * H > 0x3fffffffLL || (long long)n_tasks * Hkv > 0x3fffffffLL)
    return ZK_EINVAL;
  const SharedArgs a{q, k, v, out, part_o, part_ml, seq_start, seq_slot, page_table, words, sink, gate, status, pt_stride, n, H,
                     Hkv, hd, vd, page_size, ld_gate, scale, softcap, chunk, n_tasks, shared_splits, own_splits, own_keys, H / Hkv,
                     page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size), 0};
  if (mma_takes(dtype, H / Hkv, hd, vd, page_size)) {
    if ((uintptr_t)q % 4 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)out % 8) return ZK_EINVAL;
    const int rc = hd == 64 ? launch_rows<64>(a, tile_rows, num_pages, stream) : launch_rows<128>(a, tile_rows, num_pages, stream);
    if (rc) return rc;
    return launch_merge<bf16>(a, stream);
  }
  if ((tile_rows != 16 && tile_rows != 32) || (dtype != ZK_F32 && dtype != ZK_BF16)) return ZK_EINVAL;
  const int rc = dtype == ZK_F32 ? launch_general<float>(a, tile_rows, stream) : launch_general<bf16>(a, tile_rows, stream);
  if (rc) return rc;
  return dtype == ZK_F32 ? launch_merge<float>(a, stream) : launch_merge<bf16>(a, stream);
}

}  // extern "C"
