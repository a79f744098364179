// Copies inside the cache: the first tokens of pages, in every layer and head, and whole rows of per-sequence state.
//
// A tensor is seen as [layers, entries, heads, units] with units of `unit` bytes that lie side by side (a token's row of
// one head; a whole state row is one unit of its only head), and a move (src, dst, count) copies the first `count` units of
// entry src to entry dst in every layer and head.  No entry is written by two moves or read by one and written by
// another (checked on the host), so the order does not matter.  The moves travel as kernel parameters: nothing is
// copied to the device first, and a recorded copy keeps its own.
//
// Bound by the bytes: a block copies 16 KB of one run of units, its threads' loads all requested before the first store, and
// several copies of one entry are written from one read of it.  512 pages of 6 layers x 8 heads x 8 KB, keys and values:
// 125 us, 6.4 TB/s read and written (a plain copy of as many bytes: 6.5).  63 copies of 41 tokens and of a state of 131,072
// numbers in 6 calls: 41 us for 234 MB, nearly all of it written.
#include "common.cuh"
#include <algorithm>
#include <atomic>
#include <new>

namespace {

constexpr int MOST_MOVES = 320;       // with the tensors just under the 4 KB that kernel parameters always have
constexpr int MOST_TENSORS = 4;
constexpr int THREADS = 256, PER_THREAD = 4, PIECE = THREADS * PER_THREAD * 16;

struct Tensor {
  char* base;
  long long layer_stride, entry_stride, head_stride;   // bytes
  int layers, entries, heads, unit;
};
struct CopyArgs {
  Tensor t[MOST_TENSORS];
  int n_moves, most_count;
  int src[MOST_MOVES], dst[MOST_MOVES], count[MOST_MOVES];
};

template <typename V>
__device__ __forceinline__ void copy_bytes(char* dst, const char* src, int bytes) {
  const int n = bytes / (int)sizeof(V);
  for (int i = threadIdx.x; i < n; i += THREADS) reinterpret_cast<V*>(dst)[i] = reinterpret_cast<const V*>(src)[i];
}

// Any alignment: the widest pieces that addresses and length allow.
__device__ __forceinline__ void copy_piece(char* dst, const char* src, int bytes) {
  const unsigned long long any = (unsigned long long)src | (unsigned long long)dst | (unsigned long long)bytes;
  if (any % 16 == 0) {
    uint4 v[PER_THREAD];
#pragma unroll
    for (int u = 0; u < PER_THREAD; ++u) {
      const int at = (u * THREADS + threadIdx.x) * 16;
      if (at < bytes) v[u] = *reinterpret_cast<const uint4*>(src + at);
    }
#pragma unroll
    for (int u = 0; u < PER_THREAD; ++u) {
      const int at = (u * THREADS + threadIdx.x) * 16;
      if (at < bytes) *reinterpret_cast<uint4*>(dst + at) = v[u];
    }
  } else if (any % 4 == 0) {
    copy_bytes<unsigned>(dst, src, bytes);
  } else if (any % 2 == 0) {
    copy_bytes<unsigned short>(dst, src, bytes);
  } else {
    copy_bytes<unsigned char>(dst, src, bytes);
  }
}

// RUN 1: a block per piece and move.  RUN > 1: a block makes RUN moves after one another and reads a piece that several of them
// copy once (the moves of a fork: one entry, many copies).
template <int RUN>
__global__ void __launch_bounds__(THREADS) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
  zk_wait_prior();
  const Tensor& t = a.t[blockIdx.z];
  const int pieces = (int)(((long long)a.most_count * t.unit + PIECE - 1) / PIECE);
  const int runs = (a.n_moves + RUN - 1) / RUN;
  const long long items = (long long)t.layers * t.heads * pieces * runs;
  for (long long i = blockIdx.x; i < items; i += gridDim.x) {
    const int piece = (int)(i % pieces);
    long long j = i / pieces;
    const int m0 = (int)(j % runs) * RUN;
    j /= runs;
    const int head = (int)(j % t.heads), layer = (int)(j / t.heads);
    const long long from = (long long)piece * PIECE;
    char* base = t.base + layer * t.layer_stride + head * t.head_stride + from;
    auto bytes_of = [&](int mv) { return (int)max(0LL, min((long long)a.count[mv] * t.unit - from, (long long)PIECE)); };
    const int first = bytes_of(m0);
    if (RUN == 1) {
      if (first > 0) copy_piece(base + a.dst[m0] * t.entry_stride, base + a.src[m0] * t.entry_stride, first);
      continue;
    }
    const int m1 = min(a.n_moves, m0 + RUN);
    bool same = true;                    // one source, one length, everything on 16 bytes
    unsigned long long any = (unsigned long long)(base + a.src[m0] * t.entry_stride) | (unsigned long long)first;
    for (int mv = m0; mv < m1; ++mv) {
      same &= a.src[mv] == a.src[m0] && a.count[mv] == a.count[m0];
      any |= (unsigned long long)(base + a.dst[mv] * t.entry_stride);
    }
    if (!same || any % 16) {
      for (int mv = m0; mv < m1; ++mv)
        if (bytes_of(mv) > 0) copy_piece(base + a.dst[mv] * t.entry_stride, base + a.src[mv] * t.entry_stride, bytes_of(mv));
      continue;
    }
    const char* src = base + a.src[m0] * t.entry_stride;
    uint4 v[PER_THREAD];
#pragma unroll
    for (int u = 0; u < PER_THREAD; ++u) {
      const int at = (u * THREADS + threadIdx.x) * 16;
      if (at < first) v[u] = *reinterpret_cast<const uint4*>(src + at);
    }
    for (int mv = m0; mv < m1; ++mv) {
      char* dst = base + a.dst[mv] * t.entry_stride;
#pragma unroll
      for (int u = 0; u < PER_THREAD; ++u) {
        const int at = (u * THREADS + threadIdx.x) * 16;
        if (at < first) *reinterpret_cast<uint4*>(dst + at) = v[u];
      }
    }
  }
}

}  // namespace

// The current device's SMs, asked for once per device.
static int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 1;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

extern "C" {

// What a copy must not be given, since it would leave the tensors: 1: an entry outside; 2: a count outside.  Host only.
static int outside(const int* src, const int* dst, const int* count, int n, long long entries, int units) {
  for (int i = 0; i < n; ++i) {
    if (src[i] < 0 || dst[i] < 0 || src[i] >= entries || dst[i] >= entries) return 1;
    if (count && (count[i] < 0 || count[i] > units)) return 2;
  }
  return 0;
}

// Whether n moves among `entries` entries of `units` units are sound: 0; 1: an entry outside; 2: a count outside; 3: an entry
// written twice, or read and written; 4: no memory for the check.  Host only.
int zk_cache_moves_check(const int* src, const int* dst, const int* count, int n, int entries, int units) {
  if (const int rc = outside(src, dst, count, n, entries, units)) return rc;
  if (n <= 0) return 0;
  if (n == 1) return src[0] == dst[0] ? 3 : 0;
  int* s = new (std::nothrow) int[2 * (size_t)n];
  if (!s) return 4;
  int *d = s + n, rc = 0;
  std::copy(src, src + n, s);
  std::copy(dst, dst + n, d);
  std::sort(s, s + n);
  std::sort(d, d + n);
  for (int i = 1; i < n && !rc; ++i) rc = d[i] == d[i - 1] ? 3 : 0;
  for (int i = 0, j = 0; i < n && j < n && !rc;) {
    if (s[i] == d[j]) rc = 3;
    else if (s[i] < d[j]) ++i;
    else ++j;
  }
  delete[] s;
  return rc;
}

// `tensors` (host memory): n_tensors x 8 long long: address, layer, entry and head stride in bytes, layers, entries, heads,
// bytes of a unit.  src, dst, count (host memory): n_moves each, sound for `units` units an entry (zk_cache_moves_check; here
// only what lies outside is refused); no count: all units.  One launch for every MOST_TENSORS tensors and MOST_MOVES moves.
int zk_cache_copy(const void* tensors, int n_tensors, const int* src, const int* dst, const int* count, int n_moves, int units,
                  cudaStream_t stream) {
  if (n_moves <= 0 || n_tensors <= 0) return 0;
  if (!tensors || !src || !dst || units <= 0) return ZK_EINVAL;
  const long long* d = (const long long*)tensors;
  for (int i = 0; i < n_tensors; ++i)
    if (!d[8 * i] || d[8 * i + 4] <= 0 || d[8 * i + 5] <= 0 || d[8 * i + 6] <= 0 || d[8 * i + 7] <= 0 || d[8 * i + 7] > 0x7fffffffLL ||
        outside(src, dst, count, n_moves, d[8 * i + 5], units))
      return ZK_EINVAL;
  for (int t0 = 0; t0 < n_tensors; t0 += MOST_TENSORS)
    for (int m0 = 0; m0 < n_moves; m0 += MOST_MOVES) {
      CopyArgs a;
      const int nt = std::min(MOST_TENSORS, n_tensors - t0), nm = std::min(MOST_MOVES, n_moves - m0);
      a.n_moves = nm;
      a.most_count = 0;
      for (int i = 0; i < nm; ++i) {
        a.src[i] = src[m0 + i];
        a.dst[i] = dst[m0 + i];
        a.count[i] = count ? count[m0 + i] : units;
        a.most_count = std::max(a.most_count, a.count[i]);
      }
      if (a.most_count == 0) continue;
      long long most = 0;
      for (int i = 0; i < nt; ++i) {
        const long long* e = d + 8 * (t0 + i);
        a.t[i] = {(char*)e[0], e[1], e[2], e[3], (int)e[4], (int)e[5], (int)e[6], (int)e[7]};
        most = std::max(most, e[4] * e[6] * (((long long)a.most_count * e[7] + PIECE - 1) / PIECE));
      }
      // Runs of copies of one entry: where that still leaves four blocks per SM.  63 copies of 41 tokens and of a state of
      // 6 x 512 KB when this was chosen: 43.0 us in runs of four (43.4 of eight, 46.7 of sixteen), 47.2 one by one; 512 pages that are
      // copied once 145 and 128.
      int follow = 0;
      for (int i = 1; i < nm; ++i) follow += a.src[i] == a.src[i - 1] && a.count[i] == a.count[i - 1];
      const bool spread = 4 * follow >= 3 * (nm - 1) && most * (nm / 4) >= 4LL * sm_count();
      const dim3 grid((unsigned)std::min(most * (spread ? (nm + 3) / 4 : nm), 1LL << 30), 1, nt);
      const int rc = spread ? zk_launch_dependent(cache_copy_kernel<4>, grid, dim3(THREADS), 0, stream, a)
                            : zk_launch_dependent(cache_copy_kernel<1>, grid, dim3(THREADS), 0, stream, a);
      if (rc) return rc;
    }
  return 0;
}

}  // extern "C"
