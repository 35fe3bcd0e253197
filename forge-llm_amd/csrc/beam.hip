// Beam search (fg_beam_*): the choice of the next beams over beams and
// vocabulary, and the beams' states following their parents in place.
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBeams = 64;

// ── selection ─────────────────────────────────────────────────────────────
// Each logit is read once, so the choice is made in two launches: a workgroup
// per segment of a row leaves the segment's maximum, sum of exponentials and W
// first candidates, then a workgroup per request adds the segments' sums up and
// picks among their candidates, in fp64; the exponentials and a segment's sum are
// fp32, which leaves a row's log sum good to about 2^-20.  Both find the W first of many
// without sorting them: the W-th greatest of the threads' own maxima bounds the
// W-th greatest of all from below, few values reach it, and those are ranked by
// counting.  The segments' lists are in order, so the second launch reads each only
// as far as it reaches the bound.  Latency-bound but for large vocabularies: 1 request
// of 4 beams over 4,096 tokens 9.4 us, 8 of 8 over 128,256 17 (reading and the
// exponentials 11.6 of it, 2.8 TB/s), 1 of 32 19 (1,065 with all candidates looked
// at), 1 of 64 25 (3,992).
//
// Values are compared as unsigned keys in the order of the values: none 0, NaN
// 1, -inf the lowest number, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  return x != x ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k == 1u ? 0x7FC00000u : (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return x != x ? 1ull : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return __builtin_bit_cast(double, k == 1ull ? 0x7FF8000000000000ull
                                    : (k >> 63) ? k ^ 0x8000000000000000ull
                                                : ~k);
}

constexpr int kListed = 1024;  // candidates that are ranked by counting

// The segment's candidates beyond kListed (ties, mostly): the W-th greatest key
// and, among its equals, the place of the last one taken, bit by bit.
template <int E>
__device__ void exact_border(uint32_t& border, int& last, const uint32_t (&key)[E], int W, int* sh) {
  const int wave = threadIdx.x >> 6;
  auto count = [&](auto in) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += __popcll(__ballot(in(e)));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[wave] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kWaves; ++w) n += sh[w];
    return n;
  };
  border = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = border | (1u << bit);
    if (count([&](int e) { return key[e] >= t; }) >= W) border = t;
  }
  const int need = W - count([&](int e) { return key[e] > border; });
  // place of element e of a thread, in the order of the row
  auto place = [&](int e) { return (e >> 2) * 4 * kThreads + 4 * (int)threadIdx.x + (e & 3); };
  last = 0;  // count(place < last) < need <= count(place <= last)
  for (int bit = 14; bit >= 0; --bit) {
    const int t = last + (1 << bit);
    if (count([&](int e) { return key[e] == border && place(e) < t; }) < need) last = t;
  }
}

// Segment blockIdx.x of row blockIdx.y: up to 4 P values a thread.
template <int P>
__global__ void __launch_bounds__(kThreads) beam_segment_kernel(float2* __restrict__ sums, uint2* __restrict__ cand,
                                                                const float* __restrict__ logits, int64_t ld,
                                                                const int32_t* __restrict__ done, int W, int V,
                                                                int length) {
  constexpr int E = 4 * P;
  __shared__ uint32_t best[kThreads], bound;
  __shared__ uint64_t list[kListed];  // key << 32 | ~place: one comparison ranks two
  __shared__ float shm[kWaves], shs[kWaves];
  __shared__ int shn[kWaves], listed;
  const int64_t row = blockIdx.y;
  if (done && done[row]) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.x * length, n = min(length, V - first);
  const float* x = logits + row * ld + first;
  float v[E];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = 4 * ((int)threadIdx.x + p * kThreads);
    if (at + 4 <= n) {
      __builtin_memcpy(&v[4 * p], x + at, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * p + e] = at + e < n ? x[at + e] : -INFINITY;
    }
  }
  if (threadIdx.x == 0) listed = 0;
  float most = v[0];
#pragma unroll
  for (int e = 1; e < E; ++e) most = fmaxf(most, v[e]);
  const uint32_t mine = 4 * (int)threadIdx.x < n ? key_of(most) : 0u;
  best[threadIdx.x] = mine;
  float m = fg_wave_max(most);
  if (lane == 0) shm[wave] = m;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, shm[w]);
  if (wave == 0) {
    // the W-th greatest of the threads' maxima, its low bits dropped
    uint32_t b[kWaves], t = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) b[w] = best[w * 64 + lane];
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t u = t | (1u << bit);
      int c = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) c += __popcll(__ballot(b[w] >= u));
      if (c >= W) t = u;
    }
    if (lane == 0) bound = t;
  }
  // exp(x - m) in fp32: good to 2^-21 where it counts
  const float from = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((v[e] - from) * 1.44269504088896340736f);
  s = fg_wave_sum(s);
  if (lane == 0) shs[wave] = s;
  __syncthreads();
  uint32_t border = bound;
  const float least = value_of(border);
  // where W threads have numbers above -inf, the values from `least` on are
  // enough; else all of the segment are candidates
  const bool bounded = border > key_of(-INFINITY);
  if (!bounded || mine >= border) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = 4 * ((int)threadIdx.x + (e >> 2) * kThreads) + (e & 3);
      if (bounded ? v[e] >= least : at < n) {
        const int i = atomicAdd(&listed, 1);
        if (i < kListed) list[i] = (uint64_t)key_of(v[e]) << 32 | ~(uint32_t)at;
      }
    }
  }
  __syncthreads();
  int c = listed;
  if (c > kListed) {  // the same for all threads
    int last;
    uint32_t key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = 4 * ((int)threadIdx.x + (e >> 2) * kThreads) + (e & 3);
      key[e] = at < n ? key_of(v[e]) : 0u;
    }
    exact_border<E>(border, last, key, W, shn);
    __syncthreads();
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = 4 * ((int)threadIdx.x + (e >> 2) * kThreads) + (e & 3);
      if (key[e] > border || (key[e] == border && at <= last)) {
        const int i = atomicAdd(&listed, 1);
        if (i < kListed) list[i] = (uint64_t)key[e] << 32 | ~(uint32_t)at;
      }
    }
    __syncthreads();
    c = min(listed, kListed);
  }
  const int64_t seg = row * gridDim.x + blockIdx.x;
  cand += seg * W;
  for (int i = threadIdx.x; i < max(c, W); i += kThreads) {
    if (i >= c) {
      cand[i] = make_uint2(0u, 0u);
      continue;
    }
    const uint64_t me = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < c; ++j) rank += list[j] > me;
    if (rank < W) cand[rank] = make_uint2((uint32_t)(me >> 32), ~(uint32_t)me + first);
  }
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < kWaves; ++w) s += shs[w];
    sums[seg] = make_float2(m, s);
  }
}

// One workgroup per request.  A candidate's second key orders those of equal
// value: the lower beam, within it the greater logit, then the lower token.
constexpr int kTokenBits = 26;
constexpr int kPick = 512, kPickWaves = kPick / 64;
static_assert(kPick >= 8 * kMaxBeams, "every beam has lanes");
__global__ void __launch_bounds__(kPick) beam_pick_kernel(float* __restrict__ score_out, int32_t* __restrict__ token,
                                                             int32_t* __restrict__ parent, int32_t* __restrict__ done_out,
                                                             const float2* __restrict__ sums,
                                                             const uint2* __restrict__ cand,
                                                             const float* __restrict__ scores,
                                                             const int32_t* __restrict__ done, int eos, int W, int V,
                                                             int S) {
  __shared__ double base[kMaxBeams];
  __shared__ int kind[kMaxBeams];  // 0: its candidates, 1: all equal to base, 2: done
  __shared__ ulonglong2 list[kListed];
  __shared__ unsigned long long border[kPickWaves];
  __shared__ uint32_t best[kPick];
  __shared__ int listed;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * W;
  // W S sorted lists of W candidates, each dealt out to `m` threads (its candidates
  // r, r + m, ...), as many as there are
  const int lists = W * S, m = min(W, max(1, kPick / lists)), parts = lists * m;
  const uint2* mine = cand + r0 * lists;
  uint2 held = make_uint2(0u, 0u);  // a thread's first candidate, fetched beside the sums
  if ((int)threadIdx.x < parts) held = mine[threadIdx.x / m * W + threadIdx.x % m];
  {  // the beams' log sums, all at once: L lanes each
    const int L = W <= 8 ? 64 : W <= 16 ? 32 : W <= 32 ? 16 : 8;
    const int b = threadIdx.x / L, l = threadIdx.x & (L - 1);
    if (b < W) {
      const bool fin = done && done[r0 + b];
      const double score = scores[r0 + b];
      float most = -INFINITY;
      double s = 0.0;
      if (!fin) {
        const float2* row = sums + (r0 + b) * S;
        for (int z = l; z < S; z += L) most = fmaxf(most, row[z].x);
        for (int o = L / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        for (int z = l; z < S; z += L)
          s += (double)row[z].y *
               (row[z].x == most ? 1.f : __builtin_amdgcn_exp2f((row[z].x - most) * 1.44269504088896340736f));
        for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      }
      if (l == 0) {
        const double v = fin ? score : most == -INFINITY && s == 0.0 ? -INFINITY : score - ((double)most + log(s));
        base[b] = v;
        kind[b] = fin ? 2 : fabs(v) < INFINITY ? 0 : 1;
      }
    }
  }
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  auto candidate = [&](int l, int j, uint2 c, ulonglong2& k) {  // j of list l
    const int b = l / S, z = l - b * S;
    k = make_ulonglong2(0, 0);
    if (kind[b] == 0) {
      if (c.x == 0) return;
      k.x = key_of(base[b] + (double)value_of(c.x));
    } else if (kind[b] == 1) {
      if (z != 0 || j >= V) return;  // all equal: the first W tokens
      k.x = key_of(base[b]);
      c = make_uint2(1u, (uint32_t)j);
    } else {
      if (z != 0 || j != 0) return;
      k.x = key_of(base[b]);
      c = make_uint2(1u, (uint32_t)eos);
    }
    k.y = ((uint64_t)(kMaxBeams - 1 - b) << (32 + kTokenBits)) | ((uint64_t)c.x << kTokenBits) |
          ((1u << kTokenBits) - 1 - c.y);
  };
  auto put = [&](int rank, const ulonglong2& k) {
    const int b = kMaxBeams - 1 - (int)(k.y >> (32 + kTokenBits));
    const int t = (1 << kTokenBits) - 1 - (int)(k.y & ((1u << kTokenBits) - 1));
    score_out[r0 + rank] = (float)value_of((uint64_t)k.x);
    token[r0 + rank] = t;
    parent[r0 + rank] = b;
    if (done_out) done_out[r0 + rank] = kind[b] == 2 || t == eos;
  };
  // (both halves compared, without a branch between their loads)
  auto above = [](const ulonglong2& a, const ulonglong2& b) { return (a.x > b.x) | ((a.x == b.x) & (a.y > b.y)); };
  ulonglong2 k, first = make_ulonglong2(0, 0);
  uint64_t greatest = 0;
  if ((int)threadIdx.x < parts) {
    candidate(threadIdx.x / m, threadIdx.x % m, held, first);
    greatest = first.x;
  }
  for (int u = threadIdx.x + kPick; u < parts; u += kPick) {
    candidate(u / m, u % m, mine[u / m * W + u % m], k);
    greatest = k.x > greatest ? k.x : greatest;
  }
  // a bound that W candidates reach: for few beams the W-th greatest of a wave's
  // first candidates (the greatest of these), for more that of all threads' (their
  // high words)
  const uint32_t high = (uint32_t)(greatest >> 32);
  uint32_t bound = 0;
  if (W <= 8) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = bound | (1u << bit);
      if (__popcll(__ballot(high >= t)) >= W) bound = t;
    }
  } else {
    best[threadIdx.x] = high;
    __syncthreads();
    if (wave == 0) {
      uint32_t v[kPickWaves];
#pragma unroll
      for (int w = 0; w < kPickWaves; ++w) v[w] = best[w * 64 + lane];
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t t = bound | (1u << bit);
        int c = 0;
#pragma unroll
        for (int w = 0; w < kPickWaves; ++w) c += __popcll(__ballot(v[w] >= t));
        if (c >= W) bound = t;
      }
    }
  }
  if (lane == 0) border[wave] = (uint64_t)bound << 32;
  __syncthreads();
  uint64_t least = 1;
  for (int w = 0; w < kPickWaves; ++w) least = border[w] > least ? border[w] : least;
  // every part from its greatest on, as long as it reaches the bound
  for (int u = threadIdx.x; u < parts; u += kPick) {
    const int l = u / m;
    for (int j = u % m; j < W; j += m) {
      if (u == (int)threadIdx.x && j == u % m) k = first;
      else candidate(l, j, mine[l * W + j], k);
      if (k.x < least) break;
      const int at = atomicAdd(&listed, 1);
      if (at < kListed) list[at] = k;
    }
  }
  __syncthreads();
  const int c = listed;
  if (c <= kListed) {
    for (int i = threadIdx.x; i < c; i += kPick) {
      k = list[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < c; ++j) rank += above(list[j], k);
      if (rank < W) put(rank, k);
    }
    return;
  }
  // too many equals to list: one after the other
  ulonglong2 prev = make_ulonglong2(~0ull, ~0ull);
  for (int w = 0; w < W; ++w) {
    first = make_ulonglong2(0, 0);
    for (int i = threadIdx.x; i < lists * W; i += kPick) {
      candidate(i / W, i % W, mine[i], k);
      if (above(prev, k) && above(k, first)) first = k;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const ulonglong2 u = make_ulonglong2(__shfl_xor(first.x, o, 64), __shfl_xor(first.y, o, 64));
      if (above(u, first)) first = u;
    }
    __syncthreads();
    if (lane == 0) list[wave] = first;
    __syncthreads();
    first = list[0];
    for (int z = 1; z < kPickWaves; ++z)
      if (above(list[z], first)) first = list[z];
    if (threadIdx.x == 0) put(w, first);
    prev = first;
  }
}

// ── states ────────────────────────────────────────────────────────────────
// A thread holds one place of a part, sizeof(U) bytes of it, in every beam of the
// request: it reads what the beams take, then writes, so no second buffer and no
// order between threads is needed, and a beam that goes on from itself costs
// nothing.  HBM-bound: a parent that several beams take is fetched once and read
// again from the caches (8 beams of 12 layers, 664 MB moved: 128 us, 5.2 TB/s).
// States of one unit size share a launch.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
struct State {
  uint8_t* base;
  int64_t beam_stride, outer_stride, inner_stride, row_bytes;
  int inner, rows, first;  // first: the first of its parts among all
};
struct States {
  State s[FG_BEAM_STATES];
  int count;
};
template <typename U, int WM>
__global__ void __launch_bounds__(kThreads) beam_reorder_kernel(States all, const int32_t* __restrict__ parent,
                                                                const int32_t* __restrict__ len, int W) {
  __shared__ int64_t from[WM], end[WM], most;  // where a beam's bytes come from, how many
  int k = 0;
  while (k + 1 < all.count && (int)blockIdx.y >= all.s[k + 1].first) ++k;
  const State& s = all.s[k];
  const int64_t r0 = (int64_t)blockIdx.z * W;
  if (threadIdx.x < 64) {
    const int b = threadIdx.x;
    int p = b;
    int64_t e = 0;
    if (b < W) {
      const int q = parent[r0 + b];
      if (q >= 0 && q < W && q != b) {
        p = q;
        e = (len ? min(max(len[r0 + p], 0), s.rows) : s.rows) * s.row_bytes;
      }
    }
    if (b < WM) {
      from[b] = p * s.beam_stride;
      end[b] = e;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const int64_t u = __shfl_xor((long long)e, o, 64);
      e = u > e ? u : e;
    }
    if (b == 0) most = e;
  }
  __syncthreads();
  const int part_of = blockIdx.y - s.first;
  uint8_t* part = s.base + r0 * s.beam_stride + (part_of / s.inner) * s.outer_stride +
                  (part_of % s.inner) * s.inner_stride;
  constexpr int64_t step = sizeof(U);
  for (int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * step; at < most;
       at += (int64_t)gridDim.x * kThreads * step) {
    U v[WM];
    bool cut = false;
#pragma unroll
    for (int b = 0; b < WM; ++b) {
      if (at + step <= end[b]) v[b] = *reinterpret_cast<const U*>(part + from[b] + at);
      else cut |= at < end[b];
    }
    if (step > 2 && cut) {
      // a beam's last bytes, less than a unit, two at a time: nothing of this unit
      // has been written yet, and these two bytes of it are read before they are
      for (int64_t e = at; e < at + step; e += 2) {
        uint16_t t[WM];
#pragma unroll
        for (int b = 0; b < WM; ++b)
          if (at + step > end[b] && e < end[b]) t[b] = *reinterpret_cast<const uint16_t*>(part + from[b] + e);
#pragma unroll
        for (int b = 0; b < WM; ++b)
          if (at + step > end[b] && e < end[b])
            *reinterpret_cast<uint16_t*>(part + b * s.beam_stride + e) = t[b];
      }
    }
#pragma unroll
    for (int b = 0; b < WM; ++b)
      if (at + step <= end[b]) *reinterpret_cast<U*>(part + b * s.beam_stride + at) = v[b];
  }
}

// The states of unit size U among all (units[i] of each).
template <typename U>
int launch_reorder(const fg_beam_state* states, int count, const int* units, const int32_t* parent, const int32_t* len,
                   int nReq, int W) {
  States all{};
  int64_t parts = 0, longest = 0;
  for (int i = 0; i < count; ++i) {
    const fg_beam_state& s = states[i];
    if (units[i] != (int)sizeof(U) || s.rows == 0) continue;
    all.s[all.count++] = {(uint8_t*)s.base, s.beam_stride, s.outer_stride, s.inner_stride, s.row_bytes, s.inner, s.rows,
                          (int)parts};
    parts += (int64_t)s.outer * s.inner;
    const int64_t n = (s.row_bytes * s.rows + sizeof(U) - 1) / sizeof(U);
    longest = n > longest ? n : longest;
  }
  if (!all.count) return FG_OK;
  int64_t gx = (longest + kThreads - 1) / kThreads;
  if (gx > 4096) gx = 4096;
  const dim3 grid((unsigned)gx, (unsigned)parts, (unsigned)nReq);
#define REORDER(WM) FG_LAUNCH((beam_reorder_kernel<U, WM>), grid, dim3(kThreads), 0, all, parent, len, W)
  if (W <= 4) REORDER(4);
  else if (W <= 8) REORDER(8);
  else if (W <= 16) REORDER(16);
  else if (W <= 32) REORDER(32);
  else if constexpr (sizeof(U) <= 8) REORDER(64);  // more beams than 32 in units of up to 8 bytes
#undef REORDER
  return FG_OK;
}

}  // namespace

extern "C" int fg_beam_select(float* score_out, int32_t* token, int32_t* parent, int32_t* done_out,
                              const float* logits, int64_t ld, const float* scores, const int32_t* done, int eos,
                              int nReq, int W, int V) {
  FG_ARG_CHECK(score_out && token && parent && logits && scores, "fg_beam_select: null argument");
  FG_ARG_CHECK(nReq > 0 && V > 0 && W >= 1 && W <= kMaxBeams && nReq <= 65535 / W,
               "fg_beam_select: bad dimensions: %d requests, %d beams (1 to %d), vocabulary %d", nReq, W, kMaxBeams, V);
  FG_ARG_CHECK(ld >= V, "fg_beam_select: row stride %lld is below the vocabulary %d", (long long)ld, V);
  FG_ARG_CHECK(!done == !done_out, "fg_beam_select: done and done_out go together");
  FG_ARG_CHECK(eos < V, "fg_beam_select: eos %d outside the vocabulary %d", eos, V);
  FG_ARG_CHECK(!done || eos >= 0, "fg_beam_select: done needs eos");
  FG_ARG_CHECK(V <= 1 << kTokenBits, "fg_beam_select: vocabulary %d is above %d", V, 1 << kTokenBits);
  FG_REQUIRE_INIT();
  const int rows = nReq * W;
  fg::KProfScope prof("beam_select", 0.0, 4.0 * rows * V);
  // segments of 1024 to 8192 logits, about 1024 of them
  int64_t S = (V + 1023) / 1024, least = (V + 8191) / 8192, want = (1024 + rows - 1) / rows;
  if (S > want) S = want > least ? want : least;
  const int per = (int)((V + S - 1) / S), P = per <= 1024 ? 1 : per <= 2048 ? 2 : per <= 4096 ? 4 : 8;
  const int length = (per + 3) / 4 * 4;
  S = (V + length - 1) / length;
  fg::Workspace ws;
  const int rc = ws.get((size_t)rows * S * (sizeof(float2) + W * sizeof(uint2)));
  if (rc != FG_OK) return rc;
  float2* sums = (float2*)ws.ptr;
  uint2* cand = (uint2*)(sums + rows * S);
  const dim3 grid((unsigned)S, (unsigned)rows);
#define SEGMENT(PS) \
  FG_LAUNCH(beam_segment_kernel<PS>, grid, dim3(kThreads), 0, sums, cand, logits, ld, done, W, V, length)
  if (P == 1) SEGMENT(1);
  else if (P == 2) SEGMENT(2);
  else if (P == 4) SEGMENT(4);
  else SEGMENT(8);
#undef SEGMENT
  FG_LAUNCH(beam_pick_kernel, dim3(nReq), dim3(kPick), 0, score_out, token, parent, done_out, (const float2*)sums,
            (const uint2*)cand, scores, done, eos, W, V, (int)S);
  return FG_OK;
}

extern "C" int fg_beam_reorder(const fg_beam_state* states, int count, const int32_t* parent, const int32_t* len,
                               int nReq, int W) {
  FG_ARG_CHECK(states && parent, "fg_beam_reorder: null argument");
  FG_ARG_CHECK(count >= 1 && count <= FG_BEAM_STATES, "fg_beam_reorder: %d states, 1 to %d expected", count,
               FG_BEAM_STATES);
  FG_ARG_CHECK(nReq > 0 && nReq <= 65535 && W >= 1 && W <= kMaxBeams,
               "fg_beam_reorder: bad dimensions: %d requests, %d beams (1 to %d)", nReq, W, kMaxBeams);
  double bytes = 0.0;
  for (int i = 0; i < count; ++i) {
    const fg_beam_state& s = states[i];
    FG_ARG_CHECK(s.base, "fg_beam_reorder: state %d is null", i);
    FG_ARG_CHECK(s.outer > 0 && s.inner > 0 && (int64_t)s.outer * s.inner <= 65535 / FG_BEAM_STATES && s.rows >= 0 &&
                     s.row_bytes >= 2,
                 "fg_beam_reorder: state %d: %d x %d parts of %d rows of %lld bytes", i, s.outer, s.inner, s.rows,
                 (long long)s.row_bytes);
    FG_ARG_CHECK((((uintptr_t)s.base | s.beam_stride | s.outer_stride | s.inner_stride | s.row_bytes) & 1) == 0,
                 "fg_beam_reorder: state %d: base, strides and row bytes must be even", i);
    FG_ARG_CHECK(s.beam_stride >= 0 && s.outer_stride >= 0 && s.inner_stride >= 0,
                 "fg_beam_reorder: state %d has a negative stride", i);
    bytes += 2.0 * s.outer * s.inner * s.row_bytes * s.rows * nReq * W;
  }
  FG_REQUIRE_INIT();
  fg::KProfScope prof("beam_reorder", 0.0, bytes);
  if (W == 1) return FG_OK;
  int units[FG_BEAM_STATES];
  for (int i = 0; i < count; ++i) {
    const fg_beam_state& s = states[i];
    const uintptr_t all = (uintptr_t)s.base | s.beam_stride | s.outer_stride | s.inner_stride;
    units[i] = all % 16 == 0 && W <= 32 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  }
  const int rc = launch_reorder<u32x4>(states, count, units, parent, len, nReq, W);
  if (rc != FG_OK) return rc;
  const int rc8 = launch_reorder<u32x2>(states, count, units, parent, len, nReq, W);
  if (rc8 != FG_OK) return rc8;
  const int rc4 = launch_reorder<uint32_t>(states, count, units, parent, len, nReq, W);
  if (rc4 != FG_OK) return rc4;
  return launch_reorder<uint16_t>(states, count, units, parent, len, nReq, W);
}
