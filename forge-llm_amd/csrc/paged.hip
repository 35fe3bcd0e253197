// Paged key-value cache (fg_paged_*): storing rows with their positions' rotation,
// reading them back, and causal attention of one or more new tokens a sequence.
//
// A page holds a head's slots next to each other, so a head's slots of a page are one run of memory,
// and four neighbouring slots (pages have at least four, at multiples of four) always are.
#include "common.h"

#include <float.h>
#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ── the cache as kernels see it ───────────────────────────────────────────
struct Cache {
  int nSeq, nKV, lg, nPages, maxPages;  // pages of 2^lg slots
  void *k, *v;
  const int32_t* table;
  int32_t* len;
};
__device__ __forceinline__ int slots(const Cache& c) { return c.maxPages << c.lg; }
// New tokens of sequence s, and the slots in use before them.
__device__ __forceinline__ int new_tokens(const int32_t* count, int s, int T) {
  return count ? min(max(count[s], 0), T) : T;
}
__device__ __forceinline__ int slots_used(const Cache& c, int s) { return min(max(c.len[s], 0), slots(c)); }
// Slot j (below slots(c)) of sequence s: the row of (layer, page, kv head 0) that holds
// its values of head h at + h 2^lg, or -1 where it has no page.
__device__ __forceinline__ int64_t slot_row(const Cache& c, int layer, int s, int j) {
  const int page = c.table[(int64_t)s * c.maxPages + (j >> c.lg)];
  if ((uint32_t)page >= (uint32_t)c.nPages) return -1;
  return ((((int64_t)layer * c.nPages + page) * c.nKV) << c.lg) + (j & ((1 << c.lg) - 1));
}

// ── store and read ────────────────────────────────────────────────────────
// Values as they are stored; a rotated one comes from fp64 by way of fp32.
template <int N>
__device__ __forceinline__ void put(float* p, const float* x) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = x[i];
}
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
template <int N>
__device__ __forceinline__ void put(_Float16* p, const float* x) {
  if constexpr (N == 4) {
    f16x4 y = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    *reinterpret_cast<f16x4*>(p) = y;
  } else
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = (_Float16)x[i];
}
template <int N>
__device__ __forceinline__ void get(float* x, const float* p) {
  if constexpr (N == 4) {
    const float4 y = *reinterpret_cast<const float4*>(p);
    x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
  } else
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = p[i];
}
template <int N>
__device__ __forceinline__ void get(float* x, const _Float16* p) {
  if constexpr (N == 4) {
    const f16x4 y = *reinterpret_cast<const f16x4*>(p);
    x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
  } else
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)p[i];
}

// A workgroup takes a token.  A thread takes P pairs (4, or 1 where rows are not
// aligned or pairs do not come in fours) of every so many heads, so that it reads
// their angles once (fp64, 64 bytes for four pairs, where a head's share of a row is 32).
// HBM-bound: 8191 tokens of 32 query heads and 8 kv heads of 128 74 us (5.0 TB/s read and
// written); a token of four sequences 3.3.
template <class KV, int P>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(Cache c, int layer, int dH, float* q_out,
                                                                const float* q, const float* __restrict__ k,
                                                                const float* __restrict__ v, int64_t ld, int nH, int T,
                                                                const int32_t* __restrict__ count,
                                                                const double* __restrict__ cos_tab,
                                                                const double* __restrict__ sin_tab, int npos, int rot,
                                                                int half) {
  const int s = blockIdx.x / T, t = blockIdx.x - s * T;
  if (t >= new_tokens(count, s, T)) return;
  const int units = dH / (2 * P), each = kThreads / units, h0 = threadIdx.x / units;
  if (h0 >= each) return;
  const int pair = (threadIdx.x - h0 * units) * P;
  const int64_t pos = (int64_t)slots_used(c, s) + t, row = blockIdx.x;
  const int64_t slot = pos < slots(c) ? slot_row(c, layer, s, (int)pos) : -1;
  const bool turned = pair < rot / 2;
  const int a = turned && half ? pair : 2 * pair, b = turned && half ? pair + rot / 2 : 2 * pair + P;
  double co[P], si[P];
  if (turned) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      co[i] = pos < npos ? cos_tab[pos * (rot / 2) + pair + i] : NAN;
      si[i] = pos < npos ? sin_tab[pos * (rot / 2) + pair + i] : NAN;
    }
  }
  for (int h = h0; h < nH + 2 * c.nKV; h += each) {
    const int kv = h - nH, vh = kv - c.nKV;  // its number among the keys and values
    if (kv >= 0 && slot < 0) continue;
    const float* x = kv < 0 ? q + row * ld + (int64_t)h * dH : vh < 0 ? k + row * ld + (int64_t)kv * dH : v + row * ld + (int64_t)vh * dH;
    float lo[P], hi[P];
    get<P>(lo, x + a);
    get<P>(hi, x + b);
    if (turned && vh < 0) {
      float x0[P], x1[P];  // the pairs' first and second values
#pragma unroll
      for (int i = 0; i < P; ++i) {
        x0[i] = half ? lo[i] : 2 * i < P ? lo[2 * i] : hi[2 * i - P];
        x1[i] = half ? hi[i] : 2 * i + 1 < P ? lo[2 * i + 1] : hi[2 * i + 1 - P];
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float y0 = (float)(x0[i] * co[i] - x1[i] * si[i]), y1 = (float)(x0[i] * si[i] + x1[i] * co[i]);
        if (half) {
          lo[i] = y0;
          hi[i] = y1;
        } else {
          (2 * i < P ? lo[2 * i] : hi[2 * i - P]) = y0;
          (2 * i + 1 < P ? lo[2 * i + 1] : hi[2 * i + 1 - P]) = y1;
        }
      }
    }
    if (kv < 0) {
      float* y = q_out + (row * nH + h) * dH;
      put<P>(y + a, lo);
      put<P>(y + b, hi);
    } else {
      KV* y = (KV*)(vh < 0 ? c.k : c.v) + (slot + ((int64_t)(vh < 0 ? kv : vh) << c.lg)) * dH;
      put<P>(y + a, lo);
      put<P>(y + b, hi);
    }
  }
}

template <class KV, int N>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(Cache c, int layer, int dH, float* __restrict__ k,
                                                              float* __restrict__ v, int64_t ld, int first, int T) {
  const int s = blockIdx.x / T, j = first + (blockIdx.x - s * T);
  const int64_t slot = slot_row(c, layer, s, j), row = blockIdx.x;
  const KV* from = (const KV*)(blockIdx.y ? c.v : c.k);
  float* to = (blockIdx.y ? v : k) + row * ld;
  for (int i = threadIdx.x * N; i < c.nKV * dH; i += kThreads * N) {
    const int h = i / dH;
    float x[N] = {};
    if (slot >= 0) get<N>(x, from + (slot + ((int64_t)h << c.lg)) * dH + (i - h * dH));
    put<N>(to + i, x);
  }
}

__global__ void paged_commit_kernel(Cache c, int T, const int32_t* __restrict__ count) {
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= c.nSeq) return;
  const int used = slots_used(c, s);
  c.len[s] = used + min(new_tokens(count, s, T), slots(c) - used);
}

// ── attention ─────────────────────────────────────────────────────────────
// The rows of a kv head are the queries of its group: row t group + h is query head h
// of the group of token t.  A wave takes a tile of NT x 16 rows through steps of Keys slots
// (16 rows and 16 slots a matrix instruction), all in registers, and joins what others
// of its workgroup and of other workgroups have found of the same rows at the end.
//
// Scores are formed slots x rows and the sums values x rows, so that a lane has one
// row (lane & 15) throughout: its reference, its sum and its factors need no other
// lane, and the scores that the instruction leaves in a lane, slots 4 g .. 4 g + 3 (g = lane >> 4)
// of a sixteen, are the second operand of the sums as they are.  The first operand of
// the sums wants a value of those slots for the lane's d: rows of V come in as runs, E values of
// every slot a lane, and the instruction's 16 rows are d = E i + e, e by e.
//
// fp32 caches multiply in fp32 (16x16x4).  fp16 caches multiply as they are
// (16x16x32), q and p against them in two fp16 pieces each: 22 bits.
//
// Bound by reading the cache: each value of K and V is read once a workgroup's rows, the products
// of 32 rows take a third of the time that 16 KB of a wave's slots take to come.  A step's loads
// are issued as soon as the registers of the one before are free.  One token after 130001 (32 query
// heads on 8 of 128, fp16) 97 us, 5.5 TB/s; five of 16 sequences up to 8192 46 us (5.2 TB/s); of
// what is left the joining launch is 5 to 6.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Queries of a call: the sequences' rows, and which slots they see.
struct Span {
  int T, group, rows;  // rows of a workgroup
  int window, sinks;
  int keys, waves;  // slots of a step, and waves that share steps out
  const int32_t* count;
};
struct Steps {  // steps of slots that some of the rows of tokens t0 .. t1 see: the first `sink`, then from `low` on
  int sink, low, total;
  __device__ __forceinline__ int at(int x) const { return x < sink ? x : x - sink + low; }
};
__device__ __forceinline__ Steps steps_of(const Cache& c, const Span& q, int used, int t0, int t1) {
  const int first = used + t0, end = min(used + t1 + 1, slots(c));  // (slots(c) <= 2^30)
  Steps s;
  s.low = q.window > 0 ? min(max(first - q.window + 1, 0), end) / q.keys : 0;
  s.sink = q.window > 0 ? min((min(q.sinks, end) + q.keys - 1) / q.keys, s.low) : 0;
  // (one at least, whose slots do not exist, for windows wholly behind the room's end)
  s.total = max(s.sink + (end + q.keys - 1) / q.keys - s.low, 1);
  return s;
}

// Which part of the work a workgroup has.  Sequences are cut into pieces of `per`
// steps, as many as make about `target` workgroups of all of them, whatever their
// lengths (which are known on the device alone, so that a recorded step serves all of
// them); every wave finds its own, its lanes sharing the sequences out.
struct Part {
  int s, kvh, tile, piece, pieces, per;
  int id;         // its number; neighbours read the same slots
  int64_t first;  // workgroups of the sequences before
};
// What the workgroups leave of a sequence for the joining launch.
struct Pieces {
  int64_t first;
  int count;
};
__device__ __forceinline__ int tiles_of(const Span& q, int tokens) { return (tokens * q.group + q.rows - 1) / q.rows; }
// Workgroups go to the eight dies in turn, each with a cache of its own: `id` of `total` such that a die has a run of them.
__device__ __forceinline__ int64_t by_die(int id, int64_t total) {
  const int64_t run = (total + 7) / 8;
  return id / 8 < run ? id % 8 * run + id / 8 : total;
}
__device__ bool part_of(Part& p, const Cache& c, const Span& q, int target) {
  const int lane = threadIdx.x & 63, each = (c.nSeq + 63) / 64;
  const int from = min(lane * each, c.nSeq), to = min(from + each, c.nSeq);
  struct Load {
    int steps, tiles;
  };
  auto load = [&](int s) {
    const int n = new_tokens(q.count, s, q.T);
    return n > 0 ? Load{steps_of(c, q, slots_used(c, s), 0, n - 1).total, tiles_of(q, n)} : Load{0, 0};
  };
  const Load first = from < to ? load(from) : Load{0, 0};  // (of up to 64 sequences there are no others)
  auto sum = [&](auto what) {
    int64_t all = from < to ? what(first) : 0;
    for (int s = from + 1; s < to; ++s) all += what(load(s));
    return all;
  };
  auto of_wave = [](int64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
  };
  const int64_t work = of_wave(sum([](Load l) { return (int64_t)l.steps * l.tiles; })) * c.nKV;
  // The fewest steps that keep the workgroups, of which the last of each sequence's has fewer, to `target`: all of
  // them at once.  (A few left over for a second round: 16 sequences up to 8192 82 us, 61 so.)
  int64_t per = max((work + target - 1) / target, (int64_t)1), mine;
  auto pieces = [&](Load l) { return l.steps ? (l.steps + p.per - 1) / p.per : 0; };
  for (int turn = 0;; ++turn) {
    p.per = ((int)min(per, (int64_t)1 << 28) + q.waves - 1) / q.waves * q.waves;
    mine = sum([&](Load l) { return (int64_t)pieces(l) * l.tiles; }) * c.nKV;
    if (turn == 6) break;
    const int64_t all = of_wave(mine);
    if (all <= target || p.per >= 1 << 28) break;
    per = max(p.per * all / target, (int64_t)p.per + 1);
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t below = __shfl_up(upto, o, 64);
    if (lane >= o) upto += below;
  }
  const int64_t id = by_die(blockIdx.x, __shfl(upto, 63, 64));
  const uint64_t has = __ballot(id < upto);
  if (has == 0) return false;
  const int owner = __builtin_ctzll(has);
  p.first = __shfl(upto - mine, owner, 64);
  for (p.s = owner * each;; ++p.s) {
    const Load l = load(p.s);
    p.pieces = pieces(l);
    const int64_t here = (int64_t)p.pieces * l.tiles * c.nKV;
    if (id < p.first + here) break;
    p.first += here;
  }
  const int in_seq = (int)(id - p.first), n = new_tokens(q.count, p.s, q.T), tiles = tiles_of(q, n);
  p.id = (int)id;
  p.piece = in_seq % p.pieces;
  p.tile = in_seq / p.pieces % tiles;
  p.kvh = in_seq / p.pieces / tiles;
  return true;
}

// The two fp16 pieces of eight values, pair by pair.  The first pieces are one conversion a pair, the remainders,
// exact before they are rounded, one mixed product each (v_fma_mix takes and gives fp16) of those very halves: the
// compiler, left alone, would convert each value a second time.
__device__ __forceinline__ void two_pieces(const float (&x)[8], f16x8& hi, f16x8& lo) {
  float minus = -1.f;
  asm("" : "+s"(minus));
  u32x4 h, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * j], x[2 * j + 1]}, f16x2));
    asm("" : "+v"(pair));
    const f16x2 y = __builtin_bit_cast(f16x2, pair);
    f16x2 rest;
    rest[0] = (_Float16)__builtin_fmaf((float)y[0], minus, x[2 * j]);
    rest[1] = (_Float16)__builtin_fmaf((float)y[1], minus, x[2 * j + 1]);
    h[j] = pair;
    l[j] = __builtin_bit_cast(uint32_t, rest);
  }
  hi = __builtin_bit_cast(f16x8, h);
  lo = __builtin_bit_cast(f16x8, l);
}

// Zeros for what is not finite; whether all was.
template <int N>
__device__ __forceinline__ bool tame_halves(uint32_t (&v)[N]) {
  bool ok = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const bool low = (v[e] & 0x7C00u) != 0x7C00u, high = (v[e] & 0x7C000000u) != 0x7C000000u;
    ok &= low & high;
    v[e] &= (low ? 0xFFFFu : 0u) | (high ? 0xFFFF0000u : 0u);
  }
  return ok;
}
template <int N>
__device__ __forceinline__ bool tame_floats(float (&v)[N]) {
  bool ok = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const bool is = fabsf(v[e]) < INFINITY;
    ok &= is;
    v[e] = is ? v[e] : 0.f;
  }
  return ok;
}

// Slots of a step as a lane holds them: keys of slot i (and 16 + i), 8 (fp32: 4) values of every 32 (16) from 8 g (4 g) on;
// values of slots 4 g .. 4 g + 3 (and 16 more on), runs of E.
template <class KV, int DH>
struct Step;
template <int DH>
struct Step<_Float16, DH> {
  static constexpr int Keys = 32, Sub = 2, E = DH == 32 ? 2 : DH == 64 ? 4 : DH == 96 ? 6 : 8, Runs = DH / (16 * E);
  static constexpr float kOver = 11.f;  // p is held as 2^11 p: up to 2^4 above the reference it is below 2^15
  f16x8 k[Sub][DH / 32];
  uint32_t v[4 * Sub][Runs][E / 2];
  __device__ __forceinline__ void load_k(const _Float16* (&row)[Sub]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int u = 0; u < Sub; ++u)
#pragma unroll
      for (int b = 0; b < DH / 32; ++b) k[u][b] = *reinterpret_cast<const f16x8*>(row[u] + 32 * b + 8 * g);
  }
  __device__ __forceinline__ void load_v(const _Float16* (&row)[Sub]) {
    const int i = threadIdx.x & 15;
#pragma unroll
    for (int j = 0; j < 4 * Sub; ++j)
#pragma unroll
      for (int r = 0; r < Runs; ++r)
        __builtin_memcpy(v[j][r], __builtin_assume_aligned(row[j / 4] + (j % 4) * DH + r * 16 * E + i * E, E == 6 ? 4 : 2 * E), 2 * E);
  }
  // Slot j's values with zeros for what is not finite; whether all of them were.
  __device__ __forceinline__ bool tame(int j) {
    bool ok = true;
#pragma unroll
    for (int r = 0; r < Runs; ++r) ok &= tame_halves<E / 2>(v[j][r]);
    return ok;
  }
  // q's operand of a tile: two pieces of q 2^e, its greatest value just below 2^15
  static constexpr int kQ = DH / 32 * 2;  // 16-byte words a lane
  static __device__ __forceinline__ float pack_q(u32x4 (*to)[64], const float* q, float factor, bool on) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    float x[DH / 32][8], m = 0.f;
#pragma unroll
    for (int b = 0; b < DH / 32; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = q[32 * b + 8 * g + j];  // (loaded in any case: a branch a value would wait for each)
        x[b][j] = on ? y * factor : 0.f;
        m = fmaxf(m, fabsf(x[b][j]));
      }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const int e = m > 0.f && m < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
#pragma unroll
    for (int b = 0; b < DH / 32; ++b) {
      f16x8 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[b][j] = __builtin_amdgcn_ldexpf(x[b][j], e);
      two_pieces(x[b], hi, lo);
      to[2 * b][lane] = __builtin_bit_cast(u32x4, hi);
      to[2 * b + 1][lane] = __builtin_bit_cast(u32x4, lo);
    }
    return __builtin_amdgcn_ldexpf(1.f, -e);
  }
  __device__ __forceinline__ void scores(f32x4 (&s)[Sub], const u32x4 (*q)[64]) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < Sub; ++u) s[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < DH / 32; ++b) {
      const f16x8 hi = __builtin_bit_cast(f16x8, q[2 * b][lane]), lo = __builtin_bit_cast(f16x8, q[2 * b + 1][lane]);
#pragma unroll
      for (int u = 0; u < Sub; ++u) {
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u][b], lo, s[u], 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u][b], hi, s[u], 0, 0, 0);
      }
    }
  }
  // o += V^T p for NT tiles of rows
  template <int NT>
  __device__ __forceinline__ void sums(f32x4 (&o)[NT][DH / 16], const f32x4 (&p)[NT][Sub]) const {
    f16x8 hi[NT], lo[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = p[n][j / 4][j % 4];
      two_pieces(x, hi[n], lo[n]);
    }
#pragma unroll
    for (int r = 0; r < Runs; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = __builtin_amdgcn_perm(v[2 * j + 1][r][e / 2], v[2 * j][r][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
        const f16x8 a = __builtin_bit_cast(f16x8, w);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][r * E + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo[n], o[n][r * E + e], 0, 0, 0);
          o[n][r * E + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi[n], o[n][r * E + e], 0, 0, 0);
        }
      }
  }
};
template <int DH>
struct Step<float, DH> {
  static constexpr int Keys = 16, Sub = 1, E = DH == 32 || DH == 96 ? 2 : 4, Runs = DH / (16 * E);
  static constexpr float kOver = 0.f;
  f32x4 k[Sub][DH / 16];
  float v[4][Runs][E];
  __device__ __forceinline__ void load_k(const float* (&row)[Sub]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int b = 0; b < DH / 16; ++b) k[0][b] = *reinterpret_cast<const f32x4*>(row[0] + 16 * b + 4 * g);
  }
  __device__ __forceinline__ void load_v(const float* (&row)[Sub]) {
    const int i = threadIdx.x & 15;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < Runs; ++r)
        __builtin_memcpy(v[j][r], __builtin_assume_aligned(row[0] + j * DH + r * 16 * E + i * E, 4 * E), 4 * E);
  }
  __device__ __forceinline__ bool tame(int j) {
    bool ok = true;
#pragma unroll
    for (int r = 0; r < Runs; ++r) ok &= tame_floats<E>(v[j][r]);
    return ok;
  }
  static constexpr int kQ = DH / 16;
  static __device__ __forceinline__ float pack_q(u32x4 (*to)[64], const float* q, float factor, bool on) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < DH / 16; ++b) {
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = q[16 * b + 4 * g + j];
        x[j] = on ? y * factor : 0.f;
      }
      to[b][lane] = __builtin_bit_cast(u32x4, x);
    }
    return 1.f;
  }
  __device__ __forceinline__ void scores(f32x4 (&s)[Sub], const u32x4 (*q)[64]) const {
    const int lane = threadIdx.x & 63;
    s[0] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < DH / 16; ++b) {
      const f32x4 x = __builtin_bit_cast(f32x4, q[b][lane]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0][b][j], x[j], s[0], 0, 0, 0);
    }
  }
  template <int NT>
  __device__ __forceinline__ void sums(f32x4 (&o)[NT][DH / 16], const f32x4 (&p)[NT][Sub]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < Runs; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            o[n][r * E + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][r][e], p[n][0][j], o[n][r * E + e], 0, 0, 0);
  }
};

// Scores are in units of log 2, references are scores; a tile's reference moves where a
// score is more than kRise above it.  It starts at the lowest finite number: scores of -inf (an infinite key) are
// p = 0 against it, where -inf - -inf would be NaN.
constexpr float kRise = 4.f, kNoScore = -FLT_MAX;
__device__ __forceinline__ float over_groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
// Whether a query of position pos of sequence s sees a slot.
__device__ __forceinline__ bool sees_some(const Cache& c, const Span& q, int s, int pos) {
  const int end = min(pos + 1, slots(c)), low = q.window > 0 ? max(pos - q.window + 1, 0) : 0;
  for (int j = 0;; j = ((j >> c.lg) + 1) << c.lg) {
    if (j >= q.sinks) j = max(j, low);
    if (j >= end) return false;
    if (slot_row(c, 0, s, j) >= 0) return true;
  }
}
// What a row's values are multiplied with at the end.  Without a sum it has seen nothing, and is zeros, or scores of
// -inf alone, of which no p is a number.
__device__ __forceinline__ float one_by(float sum, const Cache& c, const Span& q, int s, int t) {
  if (__builtin_expect(sum != 0.f, 1)) return 1.f / sum;
  return sees_some(c, q, s, slots_used(c, s) + t) ? NAN : 0.f;
}

// Infinities and NaN among the values that a row sees.  A step's products spoil them: in two pieces of p inf times the second
// is NaN or of the other sign, a p that underflows gives inf 0, and what is seen by some rows alone is
// left out.  Where that has been so (a step said it, or a sum is NaN though the p are numbers) a wave goes
// over its values once more, for the rows whose p are numbers, and adds them to their sums as they are: inf p = inf for any
// p > 0.  NaN sums are set to kLost, which swallows no infinity, and are NaN again if none came.  512 tokens after 8192
// (as below) take 1.1 ms with an infinite row of V in every 16 slots, 5.1 with nothing but them, 0.16 without.
constexpr float kLost = FLT_MAX;
// Factors that bring sums to another reference: not zero, which would make NaN of an infinite sum.
__device__ __forceinline__ float factor_of(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), FLT_MIN); }
template <class KV, int DH>
__device__ __forceinline__ bool any_odd(const KV* from) {  // of a slot's values, by the wave
  bool odd = false;
#pragma unroll
  for (int d = threadIdx.x & 63; d < DH; d += 64) odd |= !(fabsf((float)from[d]) < INFINITY);
  return __any(odd);
}
// What to multiply a value that is not finite with: 1, or NaN for a p of exactly zero (a score of -inf, of an infinite key).
template <class KV, int DH>
__device__ __forceinline__ float weight_of_odd(const float* q, float factor, const KV* key) {
  if (!any_odd<KV, DH>(key)) return 1.f;
  float x = 0.f;
#pragma unroll 8
  for (int d = 0; d < DH; ++d) x = fmaf(q[d] * factor, (float)key[d], x);
  return x == -INFINITY ? NAN : 1.f;
}

// plan, part_ml, part_o: the sequences' pieces, the pieces' references and sums, and
// values, a workgroup's rows each; null: every sequence is one piece.
template <class KV, int DH, int NT>
__global__ void __launch_bounds__(kThreads, (DH == 256 ? 1 : 2)) paged_attn_kernel(Cache c, int layer, float* __restrict__ out,
                                                              const float* __restrict__ q, int nH, float factor, Span span,
                                                              int target, Pieces* __restrict__ plan,
                                                              float2* __restrict__ part_ml, float* __restrict__ part_o) {
  using S = Step<KV, DH>;
  constexpr int Keys = S::Keys, Sub = S::Sub, E = S::E, Runs = S::Runs, M = DH / 16, kRow = DH + 4;
  constexpr int kShared = NT * S::kQ * 64 * 16 > kWaves * 16 * kRow * 4 ? NT * S::kQ * 64 * 16 : kWaves * 16 * kRow * 4;
  __shared__ __attribute__((aligned(16))) uint8_t shared[kShared];  // q's operand, and the waves' values at the end
  __shared__ float2 wave_ml[kWaves][NT * 16];
  u32x4(*const qs)[64] = reinterpret_cast<u32x4(*)[64]>(shared);  // [NT kQ]
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Part p;
  if (part_ml) {
    if (!part_of(p, c, span, target)) return;
    if (p.first == p.id && threadIdx.x == 0) plan[p.s] = Pieces{p.first, p.pieces};
  } else {
    const int tiles = tiles_of(span, span.T);
    p.id = blockIdx.x;
    p.tile = blockIdx.x % tiles;
    p.kvh = blockIdx.x / tiles % c.nKV;
    p.s = blockIdx.x / tiles / c.nKV;
    if (p.s >= c.nSeq) return;
    p.piece = 0;
    p.pieces = 1;
    p.per = INT32_MAX;
  }
  const int s = __builtin_amdgcn_readfirstlane(p.s), kvh = __builtin_amdgcn_readfirstlane(p.kvh);
  const int row0 = __builtin_amdgcn_readfirstlane(p.tile) * (16 * NT), pieces = __builtin_amdgcn_readfirstlane(p.pieces);
  const int tokens = new_tokens(span.count, s, span.T), rows = min(tokens * span.group - row0, 16 * NT);
  if (rows <= 0) return;
  const int used = slots_used(c, s), t0 = row0 / span.group, t1 = (row0 + rows - 1) / span.group;
  const Steps steps = steps_of(c, span, used, t0, t1);
  const int per = __builtin_amdgcn_readfirstlane(p.per);
  const int begin = min((int64_t)__builtin_amdgcn_readfirstlane(p.piece) * per, (int64_t)steps.total);
  const int end = min((int64_t)begin + per, (int64_t)steps.total);

  // Pages of the step's slots that this lane reads: of its keys and its values.
  const int32_t* table = c.table + (int64_t)s * c.maxPages;
  struct Pages {
    int k[Sub], v[Sub];
  };
  auto find = [&](int x) {
    Pages pg;
    const int j = steps.at(min(x, steps.total - 1)) * Keys;
#pragma unroll
    for (int u = 0; u < Sub; ++u) {
      const int pk = (j + 16 * u + i) >> c.lg, pv = (j + 16 * u + 4 * g) >> c.lg;
      pg.k[u] = pk < c.maxPages ? table[pk] : -1;
      pg.v[u] = pv < c.maxPages ? table[pv] : -1;
    }
    return pg;
  };
  // Row of a slot in a layer's pages; slots of no page are read from the first page and not seen.
  const KV* const kbase = (const KV*)c.k + ((((int64_t)layer * c.nPages) * c.nKV + kvh) << c.lg) * DH;
  const KV* const vbase = (const KV*)c.v + ((((int64_t)layer * c.nPages) * c.nKV + kvh) << c.lg) * DH;
  const uint32_t inside = (1u << c.lg) - 1;
  auto row_at = [&](const KV* base, int page, int j) {
    const uint32_t there = (uint32_t)page < (uint32_t)c.nPages ? (uint32_t)page : 0u;
    return base + (((uint64_t)there * (uint32_t)c.nKV << c.lg) + ((uint32_t)j & inside)) * DH;
  };
  auto key_rows = [&](const Pages& pg, int x, const KV* (&r)[Sub]) {
    const int j = steps.at(x) * Keys;
#pragma unroll
    for (int u = 0; u < Sub; ++u) r[u] = row_at(kbase, pg.k[u], j + 16 * u + i);
  };
  auto value_rows = [&](const Pages& pg, int x, const KV* (&r)[Sub]) {
    const int j = steps.at(x) * Keys;
#pragma unroll
    for (int u = 0; u < Sub; ++u) r[u] = row_at(vbase, pg.v[u], j + 16 * u + 4 * g);
  };

  S step;
  Pages now, next;
  int x = begin + wave;
  if (x < end) {
    now = find(x);
    next = find(x + kWaves);
    const KV* r[Sub];
    key_rows(now, x, r);
    step.load_k(r);
    value_rows(now, x, r);
    step.load_v(r);
  }

  // q's operand, a wave every fourth tile of rows, and each tile's factor to the lanes
  __shared__ float unscale[NT * 16];
  for (int n = wave; n < NT; n += kWaves) {
    const int row = n * 16 + i, r = row0 + min(row, rows - 1), t = r / span.group, h = r - t * span.group;
    const float f = S::pack_q(qs + n * S::kQ, q + (((int64_t)s * span.T + t) * nH + kvh * span.group + h) * DH, factor, row < rows);
    if (g == 0) unscale[row] = f;
  }
  __syncthreads();
  float back[NT], ref[NT], sum[NT];
  int pos[NT];
  f32x4 o[NT][M];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    back[n] = unscale[n * 16 + i];
    pos[n] = used + (row0 + min(n * 16 + i, rows - 1)) / span.group;
    ref[n] = kNoScore;
    sum[n] = 0.f;
#pragma unroll
    for (int m = 0; m < M; ++m) o[n][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const int first_pos = used + t0, last_pos = used + t1;
  const int window = span.window > 0 ? span.window : INT32_MAX;
  bool odd = false;  // values that some row sees were not finite and left out of a product

  for (; x < end; x += kWaves) {
    const int j0 = steps.at(x) * Keys;
    f32x4 sc[NT][Sub];
    int again = 0;
    asm volatile("" : "+s"(again));  // q's operand is read anew each step: kept, it would fill the registers
#pragma unroll
    for (int n = 0; n < NT; ++n) step.scores(sc[n], qs + n * S::kQ + again);
    const Pages here = now;
    const bool more = x + kWaves < end;
    if (more) {
      const KV* r[Sub];
      key_rows(next, x + kWaves, r);
      step.load_k(r);
      now = next;
      next = find(x + 2 * kWaves);
    }
    bool pages = true;
#pragma unroll
    for (int u = 0; u < Sub; ++u) pages &= (uint32_t)here.v[u] < (uint32_t)c.nPages;
    // every row sees every slot of the step
    const bool whole = j0 + Keys - 1 <= first_pos && (j0 > last_pos - window || j0 + Keys <= span.sinks) && __all(pages);
    if (!whole) {
      asm volatile("");  // (a branch: most steps go past it)
      bool ok = true;
#pragma unroll
      for (int j = 0; j < 4 * Sub; ++j) {
        const int at = j0 + 16 * (j / 4) + 4 * g + j % 4;
        const bool there = (uint32_t)here.v[j / 4] < (uint32_t)c.nPages;
        ok &= step.tame(j) | !(there & (at <= last_pos) & ((at > first_pos - window) | (at < span.sinks)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bool is = there & (at <= pos[n]) & ((at > pos[n] - window) | (at < span.sinks));
          sc[n][j / 4][j % 4] = is ? sc[n][j / 4][j % 4] : -INFINITY;
        }
      }
      odd |= !__all(ok);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4 * Sub; ++j) {
        sc[n][j / 4][j % 4] *= back[n];
        top = fmaxf(top, sc[n][j / 4][j % 4]);
      }
      if (__any(top > ref[n] + kRise)) {
        const float was = ref[n];
        ref[n] = fmaxf(was, over_groups_max(top));
        const float keep = ref[n] == was ? 1.f : __builtin_amdgcn_exp2f(was - ref[n]);
        sum[n] *= keep;
#pragma unroll
        for (int m = 0; m < M; ++m) o[n][m] *= keep;
      }
      const float base = S::kOver - ref[n];
#pragma unroll
      for (int j = 0; j < 4 * Sub; ++j) {
        const float y = sc[n][j / 4][j % 4];
        float e = __builtin_amdgcn_exp2f(y + base);
        if (!whole) {
          const int at = j0 + 16 * (j / 4) + 4 * g + j % 4;
          const bool there = (uint32_t)here.v[j / 4] < (uint32_t)c.nPages;
          e = there & (at <= pos[n]) & ((at > pos[n] - window) | (at < span.sinks)) ? e : 0.f;
        }
        sum[n] += e;
        sc[n][j / 4][j % 4] = e;
      }
    }
    step.template sums<NT>(o, sc);
    if (more) {
      const KV* r[Sub];
      value_rows(now, x + kWaves, r);
      step.load_v(r);
    }
  }

  bool number[NT], lost = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sum[n] = over_groups_sum(sum[n]);
    number[n] = (n * 16 + i < rows) & (sum[n] == sum[n]);
    bool nan = odd;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) nan |= o[n][m][r] != o[n][m][r];
    lost |= number[n] & nan;
  }
  if (__builtin_expect(__any(lost), 0)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][m][r] = o[n][m][r] == o[n][m][r] ? o[n][m][r] : kLost;
    for (x = begin + wave; x < end; x += kWaves) {
      for (int j = 0; j < Keys; ++j) {
        const int at = steps.at(x) * Keys + j, page = (at >> c.lg) < c.maxPages ? table[at >> c.lg] : -1;
        if ((uint32_t)page >= (uint32_t)c.nPages) continue;
        const KV* from = row_at(vbase, page, at);
        if (!any_odd<KV, DH>(from)) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bool is = number[n] & (at <= pos[n]) & ((at > pos[n] - window) | (at < span.sinks));
          if (!__any(is)) continue;
          const int row = row0 + min(n * 16 + i, rows - 1), t = row / span.group, h = row - t * span.group;
          const float e = weight_of_odd<KV, DH>(q + (((int64_t)s * span.T + t) * nH + kvh * span.group + h) * DH, factor, row_at(kbase, page, at));
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float y = (float)from[(m / E) * 16 * E + (4 * g + r) * E + m % E];
              o[n][m][r] += (is & !(fabsf(y) < INFINITY)) ? e * y : 0.f;
              if (r == 3) __builtin_amdgcn_sched_barrier(0);  // (many at once would take registers from the common path)
            }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][m][r] = o[n][m][r] == kLost ? NAN : o[n][m][r];
  }

  // the waves' parts joined
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (g == 0) wave_ml[wave][n * 16 + i] = make_float2(ref[n], sum[n]);
  }
  float* const vals = reinterpret_cast<float*>(shared);  // [kWaves][16][kRow]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_ml[w][n * 16 + i].x);
    const float f = ref[n] == top ? 1.f : factor_of(ref[n] - top);
#pragma unroll
    for (int r = 0; r < Runs; ++r)
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int e = 0; e < E; ++e) vals[(wave * 16 + i) * kRow + r * 16 * E + (4 * g + z) * E + e] = o[n][r * E + e][z] * f;
    __syncthreads();
    constexpr int kQuads = DH / 4;
    for (int at = threadIdx.x; at < 16 * kQuads; at += kThreads) {
      const int row = at / kQuads, d = (at - row * kQuads) * 4;
      if (n * 16 + row >= rows) break;
      float most = -INFINITY, all = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) most = fmaxf(most, wave_ml[w][n * 16 + row].x);
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = wave_ml[w][n * 16 + row];
        all += ml.y * (ml.x == most ? 1.f : __builtin_amdgcn_exp2f(ml.x - most));
        y += *reinterpret_cast<const f32x4*>(vals + (w * 16 + row) * kRow + d);
      }
      if (pieces > 1) {
        const int64_t part = (int64_t)p.id * (16 * NT) + n * 16 + row;
        *reinterpret_cast<f32x4*>(part_o + part * DH + d) = y;
        if (d == 0) part_ml[part] = make_float2(most, all);
      } else {
        const int r = row0 + n * 16 + row, t = r / span.group, h = r - t * span.group;
        float* to = out + (((int64_t)s * span.T + t) * nH + kvh * span.group + h) * DH + d;
        const float f = one_by(all, c, span, s, t);
#pragma unroll
        for (int z = 0; z < 4; ++z) to[z] = y[z] * f;
      }
    }
  }
}

// ── attention of many rows ────────────────────────────────────────────────
// Where a kv head's queries fill more than a few tiles the products bound: a workgroup takes
// 128 rows, a wave 32 of them, and its waves share steps of 64 slots (fp32: 32) through LDS,
// fetched a step ahead.  32x32 instructions (16 and 2 values deep), scores slots x rows as above: a lane has
// row lane & 31 and slots 8 a + 4 h + b (h = lane >> 5; a, b < 4) of every 32, which again is the order that the sums want p in.
//
// In LDS, in words of 16 bytes:
//   K  row by row, word w of slot j at w ^ (j's swizzle): 16 slots' same word lie in different banks;
//      copied there straight from memory
//   V  the values of d at eight slots (fp32: four) that a lane's operand takes, [e][8 groups of slots][i] for d = E i + e:
//      turned around on the way, four rows of a run of E values a lane
//
// Bound by the matrix pipes: 512 tokens after 8192 (32 query heads on 8 of 128, fp16) 154 to 162 us back to back, the joining
// launch (8) among them, for 142 GFLOP of fp16 products (two pieces each): 0.9 PFLOP/s where a large library product of fp16
// matrices reaches 1.15.  (160 to 172 a launch under the tracer, where the clock settles lower.)  Two workgroups of a
// CU take turns at scores and exponentials (46% of the cycles have a matrix instruction running, 40% a vector
// one); registers (244) leave no room to interleave the two in one wave.  Every spill cost a wait for all loads: 12 of them 40 us.
template <class KV, int DH>
struct Wide;
template <int DH>
struct Wide<_Float16, DH> {
  static constexpr int Keys = 64, Sub = 2, Words = DH / 8, Quads = 2;  // quads of rows a lane turns around
  static constexpr int Lanes = DH % 64 == 0 ? 32 : 16, E = DH / Lanes, M = DH / 32;
  static constexpr float kOver = 11.f;
  f16x8 qh[DH / 16], ql[DH / 16];
  uint32_t v[8][E / 2];
  // slots of the quads that lane `lane` of wave `wave` turns around, and their group
  static __device__ __forceinline__ int group_at(int wave, int lane) { return Lanes == 32 ? 2 * wave + (lane >> 5) : 4 * wave + (lane >> 4); }
  static __device__ __forceinline__ int slot_at(int group, int quad) { return 16 * (group >> 1) + 8 * quad + 4 * (group & 1); }
  static __device__ __forceinline__ bool turns(int wave) { return Lanes == 32 || wave < 2; }
  __device__ __forceinline__ float load_q(const float* q, float factor, bool on) {
    const int h = (threadIdx.x & 63) >> 5;
    float m = 0.f;
    float x[DH / 16][8];
#pragma unroll
    for (int b = 0; b < DH / 16; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = q[16 * b + 8 * h + j];
        x[b][j] = on ? y * factor : 0.f;
        m = fmaxf(m, fabsf(x[b][j]));
      }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const int e = m > 0.f && m < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
#pragma unroll
    for (int b = 0; b < DH / 16; ++b) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[b][j] = __builtin_amdgcn_ldexpf(x[b][j], e);
      two_pieces(x[b], qh[b], ql[b]);
    }
    return __builtin_amdgcn_ldexpf(1.f, -e);
  }
  // the scores of slots 32 u .. from the rows' words
  __device__ __forceinline__ void product(f32x16& s, int b, u32x4 word) const {
    const f16x8 k = __builtin_bit_cast(f16x8, word);
    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[b], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[b], s, 0, 0, 0);
  }
  struct Probs {
    f16x8 hi[2], lo[2];
    __device__ __forceinline__ void take(const f32x16& p) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = p[8 * z + j];
        two_pieces(x, hi[z], lo[z]);
      }
    }
    // o += the word's slots
    __device__ __forceinline__ void sum(f32x16& o, int z, u32x4 word) const {
      const f16x8 a = __builtin_bit_cast(f16x8, word);
      o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, lo[z], o, 0, 0, 0);
      o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, hi[z], o, 0, 0, 0);
    }
  };
  static constexpr int Z = 2;  // words of 32 slots that a lane's operand takes
  __device__ __forceinline__ u32x4 turned(int e) const {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
    return w;
  }
  // Row j's run with zeros for what is not finite; whether all of it was.
  __device__ __forceinline__ bool tame(int j) { return tame_halves<E / 2>(v[j]); }
};
template <int DH>
struct Wide<float, DH> {
  static constexpr int Keys = 32, Sub = 1, Words = DH / 4, Quads = 1;
  static constexpr int Lanes = 32, E = DH / 32, M = DH / 32;
  static constexpr float kOver = 0.f;
  f32x4 q4[DH / 8];
  float v[4][E];
  static __device__ __forceinline__ int group_at(int wave, int lane) { return 2 * wave + (lane >> 5); }
  static __device__ __forceinline__ int slot_at(int group, int) { return 4 * group; }
  static __device__ __forceinline__ bool turns(int) { return true; }
  __device__ __forceinline__ float load_q(const float* q, float factor, bool on) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int b = 0; b < DH / 8; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = q[8 * b + 4 * h + j];
        q4[b][j] = on ? y * factor : 0.f;
      }
    return 1.f;
  }
  __device__ __forceinline__ void product(f32x16& s, int b, u32x4 word) const {
    const f32x4 k = __builtin_bit_cast(f32x4, word);
#pragma unroll
    for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], q4[b][j], s, 0, 0, 0);
  }
  struct Probs {
    f32x16 p;
    __device__ __forceinline__ void take(const f32x16& x) { p = x; }
    __device__ __forceinline__ void sum(f32x16& o, int z, u32x4 word) const {
      const f32x4 a = __builtin_bit_cast(f32x4, word);
#pragma unroll
      for (int j = 0; j < 4; ++j) o = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], p[4 * z + j], o, 0, 0, 0);
    }
  };
  static constexpr int Z = 4;
  __device__ __forceinline__ u32x4 turned(int e) const {
    const f32x4 w = {v[0][e], v[1][e], v[2][e], v[3][e]};
    return __builtin_bit_cast(u32x4, w);
  }
  __device__ __forceinline__ bool tame(int j) { return tame_floats<E>(v[j]); }
};

// 16 bytes a lane from `from` + `offset` to LDS at `lds` + 16 lane; waited for by hand (the compiler does not count
// it, which makes its own waits longer, never shorter).  m0 is given back: it cannot be named as changed; the
// scalar registers may come from a vector instruction just before, which a load has to follow by five.
__device__ __forceinline__ void load_to_lds(uint32_t lds, const void* from, uint32_t offset) {
  const uint64_t at = (uint64_t)from;
  const uint32_t high = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)), low = __builtin_amdgcn_readfirstlane((uint32_t)at);
  const uint64_t base = (uint64_t)high << 32 | low;
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(m0)
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base)
               : "memory");
}

constexpr int kWideRows = 32 * kWaves;
template <class KV, int DH>
__global__ void __launch_bounds__(kThreads, (DH == 256 ? 1 : 2)) paged_wide_kernel(
    Cache c, int layer, float* __restrict__ out, const float* __restrict__ q, int nH, float factor, Span span, int target,
    Pieces* __restrict__ plan, float2* __restrict__ part_ml, float* __restrict__ part_o) {
  using W = Wide<KV, DH>;
  constexpr int Keys = W::Keys, Sub = W::Sub, Words = W::Words, E = W::E, M = W::M, Z = W::Z, Lanes = W::Lanes;
  constexpr int kTile = Keys * Words;  // words of a step's K, and of its V
  // slot j's swizzle: the words of 16 neighbouring slots in 16 different places of 256 bytes
  constexpr int kShift = Words % 16 == 0 ? 0 : Words % 8 == 0 ? 1 : 2, kMask = Words % 16 == 0 ? 15 : Words % 8 == 0 ? 7 : 3;
  __shared__ __attribute__((aligned(16))) u32x4 lds[4 * kTile];  // [2][K, V][kTile]
  // Of a step's quads of slots: their pages, -1 for none, and whether all have one.  Pages are read up to the
  // end of their step, and those of the next but one are written in it.
  __shared__ int pages[3][Keys / 4], all_pages[3];
  __shared__ int odd_values;  // values that some row sees were not finite and left out of a product
  const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Part p;
  if (part_ml) {
    if (!part_of(p, c, span, target)) return;
    if (p.first == p.id && threadIdx.x == 0) plan[p.s] = Pieces{p.first, p.pieces};
  } else {
    const int tiles = tiles_of(span, span.T);
    // A head's tiles, which read the same slots, on one die; many heads go to the dies in turn, since sequences differ: 28
    // of up to 164 tokens, 36 heads on 12 of 128, 77 us, 91 with neighbours on a die.
    const int64_t id = c.nSeq * c.nKV >= 64 ? (blockIdx.x / 8 / tiles * 8 + blockIdx.x % 8) * tiles + blockIdx.x / 8 % tiles
                                             : by_die(blockIdx.x, (int64_t)c.nSeq * c.nKV * tiles);
    p.id = (int)id;
    // the longest first, and beside them, as the second of a CU, the shortest: 2048 tokens of 8 heads, none before them,
    // 105 us (cut into equal pieces 139)
    const int at = p.id % tiles, half = (tiles + 1) / 2;
    p.tile = at < half ? tiles - 1 - at : at - half;
    p.kvh = p.id / tiles % c.nKV;
    p.s = p.id / tiles / c.nKV;
    if (p.s >= c.nSeq) return;
    p.piece = 0;
    p.pieces = 1;
    p.per = INT32_MAX;
  }
  const int s = __builtin_amdgcn_readfirstlane(p.s), kvh = __builtin_amdgcn_readfirstlane(p.kvh);
  const int part_id = __builtin_amdgcn_readfirstlane(p.id);
  const int row0 = __builtin_amdgcn_readfirstlane(p.tile) * kWideRows, pieces = __builtin_amdgcn_readfirstlane(p.pieces);
  const int tokens = new_tokens(span.count, s, span.T), rows = min(tokens * span.group - row0, kWideRows);
  if (rows <= 0) return;
  const int used = slots_used(c, s), t0 = row0 / span.group, t1 = (row0 + rows - 1) / span.group;
  const Steps steps = steps_of(c, span, used, t0, t1);
  const int per = __builtin_amdgcn_readfirstlane(p.per);
  const int begin = min((int64_t)__builtin_amdgcn_readfirstlane(p.piece) * per, (int64_t)steps.total);
  const int end = min((int64_t)begin + per, (int64_t)steps.total);
  const int first_pos = used + t0, last_pos = used + t1;
  const int window = span.window > 0 ? span.window : INT32_MAX;

  const int32_t* table = c.table + (int64_t)s * c.maxPages;
  const KV* const kbase = (const KV*)c.k + ((((int64_t)layer * c.nPages) * c.nKV + kvh) << c.lg) * DH;
  const KV* const vbase = (const KV*)c.v + ((((int64_t)layer * c.nPages) * c.nKV + kvh) << c.lg) * DH;
  const uint32_t inside = (1u << c.lg) - 1;
  auto row_at = [&](const KV* base, int page, int j) {
    const uint32_t there = page < 0 ? 0u : (uint32_t)page;
    return base + (((uint64_t)there * (uint32_t)c.nKV << c.lg) + ((uint32_t)j & inside)) * DH;
  };
  auto page_at = [&](int x) {  // of quad threadIdx.x of step x
    const int at = (steps.at(x) * Keys + 4 * (int)threadIdx.x) >> c.lg, page = at < c.maxPages ? table[at] : -1;
    return (uint32_t)page < (uint32_t)c.nPages ? page : -1;
  };
  auto put_pages = [&](int page, int b) {
    if (threadIdx.x < Keys / 4) {
      pages[b][threadIdx.x] = page;
      const uint64_t there = __ballot(page >= 0);
      if (threadIdx.x == 0) all_pages[b] = __builtin_popcountll(there) == Keys / 4;
    }
  };
  W w;
  // Where a wave's 64 words are whole slots of a quad their page is the wave's, and they are copied straight to
  // LDS; smaller heads go through registers.
  constexpr bool kStraight = Words % 16 == 0;
  constexpr int kFetch = kTile / kThreads;
  u32x4 kw[kStraight ? 1 : kFetch];
  auto fetch_k = [&](int x, int b, int pb) {
    const int j0 = steps.at(x) * Keys;
    if constexpr (kStraight) {
      // kRows slots a load; the swizzle's bits from a load's number and a lane's part do not meet
      constexpr int kRows = 64 / Words;
      const int j = lane / Words;
      uint32_t offset = (j * Words + (lane - j * Words ^ (wave * kRows + j))) * 16;
      asm volatile("" : "+v"(offset));  // (one register, not one a load)
      int page[kFetch];
#pragma unroll
      for (int z = 0; z < kFetch; ++z) page[z] = pages[pb][(z * kWaves + wave) * kRows / 4];
#pragma unroll
      for (int z = 0; z < kFetch; ++z) {
        const int jw = (z * kWaves + wave) * kRows;  // the wave's first slot
        const KV* from = row_at(kbase, __builtin_amdgcn_readfirstlane(page[z]), j0 + jw);
        load_to_lds(lds_at + (2 * b * kTile + (z * kWaves + wave) * 64) * 16, from, offset ^ (z * kWaves * kRows & 15) * 16);
      }
    } else {
#pragma unroll
      for (int z = 0; z < kFetch; ++z) {
        const int word = (z * kWaves + wave) * 64 + lane, j = word / Words, at = (word - j * Words) ^ (j >> kShift & kMask);
        kw[z] = *reinterpret_cast<const u32x4*>(row_at(kbase, pages[pb][j / 4], j0 + j) + at * (16 / sizeof(KV)));
      }
    }
  };
  auto put_k = [&](int b) {
    if constexpr (!kStraight)
#pragma unroll
      for (int z = 0; z < kFetch; ++z) lds[2 * b * kTile + (z * kWaves + wave) * 64 + lane] = kw[z];
  };
  const int group = W::group_at(wave, lane), run = lane & (Lanes - 1);
  auto fetch_v = [&](int x, int pb) {
    if (!W::turns(wave)) return;
    const int j0 = steps.at(x) * Keys;
#pragma unroll
    for (int u = 0; u < W::Quads; ++u) {
      const int j = W::slot_at(group, u);
      const KV* from = row_at(vbase, pages[pb][j / 4], j0 + j) + run * E;
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_memcpy(w.v[4 * u + r], __builtin_assume_aligned(from + r * DH, E * sizeof(KV) % 16 == 0 ? 16 : E * sizeof(KV) % 8 == 0 ? 8 : 4), E * sizeof(KV));
    }
  };
  // Whether every row of the workgroup sees every slot of step x.
  auto is_whole = [&](int x, int pb) {
    const int j0 = steps.at(x) * Keys;
    return j0 + Keys - 1 <= first_pos && (j0 > last_pos - window || j0 + Keys <= span.sinks) && all_pages[pb] != 0;
  };
  auto put_v = [&](int x, int b, int pb) {
    if (!W::turns(wave)) return;
    if (!is_whole(x, pb)) {
      // Not every row sees all of it: what is not finite would reach, times a p of zero, rows that do not.  It becomes
      // zeros and, if any row sees it, is told of.
      bool ok = true;
      const int j0 = steps.at(x) * Keys;
#pragma unroll
      for (int u = 0; u < W::Quads; ++u) {
        const int j = W::slot_at(group, u);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = j0 + j + r;
          const bool seen = (pages[pb][j / 4] >= 0) & (at <= last_pos) & ((at > first_pos - window) | (at < span.sinks));
          ok &= w.tame(4 * u + r) | !seen;
        }
      }
      if (!ok) odd_values = 1;
    }
    u32x4* to = lds + (2 * b + 1) * kTile + group * Lanes + run;
#pragma unroll
    for (int e = 0; e < E; ++e) to[e * 8 * Lanes] = w.turned(e);
  };

  if (threadIdx.x == 0) odd_values = 0;
  if (begin < end) {
    put_pages(threadIdx.x < Keys / 4 ? page_at(begin) : -1, 0);
    __syncthreads();
    fetch_k(begin, 0, 0);
    fetch_v(begin, 0);
    if (begin + 1 < end) put_pages(threadIdx.x < Keys / 4 ? page_at(begin + 1) : -1, 1);
  }
  // the wave's rows; a wave without any computes nothing
  const int mine = min(rows - 32 * wave, 32);
  const int row = row0 + 32 * wave + min(r32, max(mine, 1) - 1);
  const int t = min(row / span.group, tokens - 1), head = kvh * span.group + (row - row / span.group * span.group);
  const int pos = used + t, wave_first = used + (row0 + 32 * wave) / span.group, wave_last = used + (row0 + 32 * wave + max(mine, 1) - 1) / span.group;
  const float back = w.load_q(q + (((int64_t)s * span.T + t) * nH + head) * DH, factor, mine > 0 && r32 < mine);
  float ref = kNoScore, sum = 0.f;
  f32x16 o[M];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int z = 0; z < 16; ++z) o[m][z] = 0.f;
  if (begin < end) {
    put_k(0);
    put_v(begin, 0, 0);
  }

  int this_page = 0;
  for (int x = begin; x < end; ++x) {
    const int b = (x - begin) & 1, j0 = steps.at(x) * Keys;
    const int next_page = this_page == 2 ? 0 : this_page + 1, free_page = 3 - this_page - next_page;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int page = -1;
    if (x + 1 < end) {
      fetch_k(x + 1, b ^ 1, next_page);
      fetch_v(x + 1, next_page);
      if (x + 2 < end && threadIdx.x < Keys / 4) page = page_at(x + 2);
    }
    const bool whole = all_pages[this_page] != 0 && j0 + Keys - 1 <= wave_first && (j0 > wave_last - window || j0 + Keys <= span.sinks);
    const bool some = mine > 0 && j0 <= wave_last && (j0 + Keys - 1 > wave_first - window || j0 < span.sinks);
    if (some) {
      const u32x4 *kt = lds + 2 * b * kTile, *vt = kt + kTile;
      // 32 slots at a time: their scores and p are all that a wave holds.  Words of K are read while the slots before
      // them are summed, the first words of V while p is formed (read when they are wanted, the waits took a third
      // of the time; all of them ahead would not fit the registers).
      constexpr int kKeyWords = Words / 2, kAhead = kKeyWords < 4 ? kKeyWords : 4;
      // word 2 k + h of slot 32 u + r32 at its swizzle: that of k = 0 with k's bits turned
      auto first_key = [&](int u) {
        const int j = 32 * u + r32;
        int word = j * Words + (h ^ (j >> kShift & kMask));
        asm volatile("" : "+v"(word));  // (the others are computed where they are read: kept, they would fill the registers)
        return word;
      };
      auto key_word = [&](int word, int k) {
        constexpr int kTurn = kMask & ~1;
        return kt[(word ^ (2 * k & kTurn)) + (2 * k & ~kTurn)];
      };
      auto value_word = [&](int u, int i) {  // of o[i % M]
        const int m = i % M, g8 = 2 * (Z * u + i / M) + h;
        return vt[Lanes == 32 ? (m * 8 + g8) * 32 + r32 : ((2 * m + (r32 >> 4)) * 8 + g8) * 16 + (r32 & 15)];
      };
      u32x4 ks[kAhead], vs[M];
      int first = first_key(0);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) ks[k] = key_word(first, k);
#pragma unroll
      for (int u = 0; u < Sub; ++u) {
        __builtin_amdgcn_sched_barrier(0);
        f32x16 sc;
#pragma unroll
        for (int z = 0; z < 16; ++z) sc[z] = 0.f;
#pragma unroll
        for (int k = 0; k < kKeyWords; ++k) {
          w.product(sc, k, ks[k % kAhead]);
          if (k + kAhead < kKeyWords) ks[k % kAhead] = key_word(first, k + kAhead);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < M; ++m) vs[m] = value_word(u, m);
        uint32_t seen = 0;  // this lane's scores
        if (!whole) {
          asm volatile("");  // (a branch: most steps go past it)
#pragma unroll
          for (int z = 0; z < 16; ++z) {
            const int j = 32 * u + 8 * (z / 4) + 4 * h + z % 4, at = j0 + j;
            const bool is = (pages[this_page][j / 4] >= 0) & (at <= pos) & ((at > pos - window) | (at < span.sinks));
            seen |= is ? 1u << z : 0u;
            sc[z] = is ? sc[z] : -INFINITY;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int z = 0; z < 16; ++z) top = fmaxf(top, sc[z]);
        top *= back;
        if (__any(top > ref + kRise)) {
          const float was = ref;
          ref = fmaxf(was, fmaxf(top, __shfl_xor(top, 32, 64)));
          const float keep = ref == was ? 1.f : __builtin_amdgcn_exp2f(was - ref);
          sum *= keep;
#pragma unroll
          for (int m = 0; m < M; ++m) o[m] *= keep;
        }
        const float base = W::kOver - ref;
#pragma unroll
        for (int z = 0; z < 16; ++z) {
          sc[z] = __builtin_amdgcn_exp2f(fmaf(sc[z], back, base));
        }
        if (!whole) {
          asm volatile("");
#pragma unroll
          for (int z = 0; z < 16; ++z) sc[z] = seen >> z & 1 ? sc[z] : 0.f;
        }
#pragma unroll
        for (int z = 0; z < 16; ++z) sum += sc[z];
        typename W::Probs pr;
        pr.take(sc);
        __builtin_amdgcn_sched_barrier(0);
        if (u + 1 < Sub) {
          first = first_key(u + 1);
#pragma unroll
          for (int k = 0; k < kAhead; ++k) ks[k] = key_word(first, k);
        }
#pragma unroll
        for (int i = 0; i < M * Z; ++i) {
          pr.sum(o[i % M], i / M, vs[i % M]);
          if (i + M < M * Z) vs[i % M] = value_word(u, i + M);
        }
      }
    }
    if (x + 1 < end) {
      put_k(b ^ 1);
      put_v(x + 1, b ^ 1, next_page);
      if (x + 2 < end) put_pages(page, free_page);
    }
    this_page = next_page;
  }
  // (found again rather than kept through the loop)
  int me = threadIdx.x;
  asm volatile("" : "+v"(me));
  const int my_row = me & 31, my_h = me >> 5 & 1, at_row = row0 + 32 * wave + my_row;
  sum += __shfl_xor(sum, 32, 64);
  auto column = [&](int m, int z) {  // of o[m][z]
    const int r = 8 * (z / 4) + 4 * my_h + z % 4;
    return Lanes == 32 ? r * E + m : (r & 15) * E + 2 * m + (r >> 4);
  };
  const bool number = (my_row < mine) & (sum == sum);
  bool lost = begin < end && odd_values != 0;  // (last written before the last step's barrier)
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int z = 0; z < 16; ++z) lost |= o[m][z] != o[m][z];
  if (__builtin_expect(__any(number & lost), 0)) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int z = 0; z < 16; ++z) o[m][z] = o[m][z] == o[m][z] ? o[m][z] : kLost;
    const int r = row0 + 32 * wave + min(my_row, mine - 1), t = r / span.group, at_pos = used + t;
    const float* const q_row = q + (((int64_t)s * span.T + t) * nH + kvh * span.group + (r - t * span.group)) * DH;
    for (int x = begin; x < end; ++x)
      for (int j = 0; j < Keys; ++j) {
        const int at = steps.at(x) * Keys + j, page = (at >> c.lg) < c.maxPages ? table[at >> c.lg] : -1;
        if ((uint32_t)page >= (uint32_t)c.nPages) continue;
        const KV* from = row_at(vbase, page, at);
        if (!any_odd<KV, DH>(from)) continue;
        const bool is = number & (at <= at_pos) & ((at > at_pos - window) | (at < span.sinks));
        if (!__any(is)) continue;
        const float e = weight_of_odd<KV, DH>(q_row, factor, row_at(kbase, page, at));
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int z = 0; z < 16; ++z) {
            const float y = (float)from[column(m, z)];
            o[m][z] += (is & !(fabsf(y) < INFINITY)) ? e * y : 0.f;
            if (z % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (many at once would take registers from the common path)
          }
      }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int z = 0; z < 16; ++z) o[m][z] = o[m][z] == kLost ? NAN : o[m][z];
  }
  if (my_row >= mine) return;
  const int64_t part = (int64_t)part_id * kWideRows + 32 * wave + my_row;
  const int my_t = at_row / span.group, my_head = kvh * span.group + (at_row - my_t * span.group);
  const float f = pieces > 1 ? 1.f : one_by(sum, c, span, s, my_t);
  float* const to = pieces > 1 ? part_o + part * DH : out + (((int64_t)s * span.T + my_t) * nH + my_head) * DH;
  if (pieces > 1 && my_h == 0) part_ml[part] = make_float2(ref, sum);
#pragma unroll
  for (int z = 0; z < 16; ++z)
#pragma unroll
    for (int m = 0; m < M; ++m) to[column(m, z)] = o[m][z] * f;
}

// A workgroup joins the pieces of R rows of a kv head, R <= kThreads / (DH / 4): its threads share out quads of a
// row's values, the rows, and (a set of threads each) the pieces, four pieces in flight.
template <int DH>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(Cache c, float* __restrict__ out, int nH, Span span, int R,
                                                              const Pieces* __restrict__ plan,
                                                              const float2* __restrict__ part_ml,
                                                              const float* __restrict__ part_o) {
  constexpr int kQuads = DH / 4, kLanes = kThreads / kQuads, kAtOnce = 4;
  __shared__ f32x4 vals[kLanes][kQuads];
  __shared__ float2 mls[kLanes];
  const int blocks = (span.T * span.group + R - 1) / R;
  const int s = blockIdx.x / blocks / c.nKV, kvh = blockIdx.x / blocks % c.nKV, row0 = blockIdx.x % blocks * R;
  const Pieces p = plan[s];  // (of no tokens: whatever was there, and not used)
  const int tokens = new_tokens(span.count, s, span.T), rows = min(tokens * span.group - row0, R);
  if (rows <= 0 || p.count <= 1) return;
  const int sets = kLanes / R, lane = threadIdx.x / kQuads, quad = threadIdx.x - lane * kQuads, set = lane / R;
  const int mine = lane - set * R, row = row0 + mine, tile = row / span.rows;
  const bool on = lane < kLanes && set < sets && mine < rows;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, all = 0.f;
  // what a piece adds, its reference brought to the greatest so far
  auto add = [&](float2 ml, f32x4 v) {
    const float was = top;
    top = fmaxf(top, ml.x);
    const float keep = was == top ? 1.f : factor_of(was - top), f = ml.x == top ? 1.f : factor_of(ml.x - top);
    all = all * keep + ml.y * f;
    y = y * keep + v * f;
  };
  if (on) {
    const int64_t first = (p.first + ((int64_t)kvh * tiles_of(span, tokens) + tile) * p.count) * span.rows + (row - tile * span.rows);
    for (int x0 = set; x0 < p.count; x0 += kAtOnce * sets) {
      float2 ml[kAtOnce];
      f32x4 v[kAtOnce];
#pragma unroll
      for (int z = 0; z < kAtOnce; ++z) {
        const int64_t at = first + (int64_t)min(x0 + z * sets, p.count - 1) * span.rows;
        ml[z] = part_ml[at];
        v[z] = *reinterpret_cast<const f32x4*>(part_o + at * DH + 4 * quad);
      }
#pragma unroll
      for (int z = 0; z < kAtOnce; ++z)
        if (x0 + z * sets < p.count) add(ml[z], v[z]);
    }
  }
  if (sets > 1) {
    if (lane < kLanes) {
      vals[lane][quad] = y;
      if (quad == 0) mls[lane] = make_float2(top, all);
    }
    __syncthreads();
    if (set == 0 && on)
      for (int x = 1; x < sets; ++x) add(mls[lane + x * R], vals[lane + x * R][quad]);
  }
  if (!on || set != 0) return;
  const int t = row / span.group, h = kvh * span.group + (row - t * span.group);
  const float f = one_by(all, c, span, s, t);
  float* to = out + (((int64_t)s * span.T + t) * nH + h) * DH + 4 * quad;
#pragma unroll
  for (int z = 0; z < 4; ++z) to[z] = y[z] * f;
}

// ── entry points' checks ──────────────────────────────────────────────────
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int check_step(const fg_paged_cache* c, int layer, int T, const char* fn) {
  FG_ARG_CHECK(layer >= 0 && layer < c->nLayers, "%s: layer %d outside [0, %d)", fn, layer, c->nLayers);
  FG_ARG_CHECK(T >= 0, "%s: T %d is negative", fn, T);
  FG_ARG_CHECK((int64_t)c->nSeq * T <= INT32_MAX / kThreads, "%s: %d sequences x %d tokens are too many", fn, c->nSeq, T);
  return FG_OK;
}
Cache view(const fg_paged_cache* c) {
  return {c->nSeq, c->nKvHeads, __builtin_ctz(c->pageSize), c->nPages, c->maxPages, c->k, c->v, c->table, c->len};
}
double row_bytes(const fg_paged_cache* c) { return (double)c->nKvHeads * c->dHead * (c->type ? 2 : 4); }

}  // namespace

int fg::check_paged_cache(const fg_paged_cache* c, const char* fn) {
  FG_ARG_CHECK(c, "%s: null cache", fn);
  FG_ARG_CHECK(c->nLayers > 0 && c->nSeq > 0 && c->nKvHeads > 0 && c->nPages > 0 && c->maxPages > 0,
               "%s: bad dimensions: %d layers, %d sequences, %d kv heads, %d pages, %d a sequence", fn, c->nLayers,
               c->nSeq, c->nKvHeads, c->nPages, c->maxPages);
  const int d = c->dHead, p = c->pageSize;
  FG_ARG_CHECK(d == 32 || d == 64 || d == 96 || d == 128 || d == 256,
               "%s: head size %d is not one of 32, 64, 96, 128, 256", fn, d);
  FG_ARG_CHECK(p >= 4 && p <= 1024 && (p & (p - 1)) == 0, "%s: page size %d is not a power of two from 4 to 1024", fn, p);
  FG_ARG_CHECK((int64_t)c->maxPages * p <= 1 << 30, "%s: %d pages of %d slots a sequence are above 2^30", fn,
               c->maxPages, p);
  FG_ARG_CHECK(c->nKvHeads <= 1 << 16 && (int64_t)c->nLayers * c->nPages < (int64_t)1 << 36,
               "%s: %d layers of %d pages of %d kv heads are too many", fn, c->nLayers, c->nPages, c->nKvHeads);
  FG_ARG_CHECK(c->type == 0 || c->type == 1, "%s: type %d is neither F32 (0) nor F16 (1)", fn, c->type);
  FG_ARG_CHECK(c->k && c->v && c->table && c->len, "%s: null array", fn);
  FG_ARG_CHECK(aligned16(c->k) && aligned16(c->v), "%s: the cache's pages must be 16-byte aligned", fn);
  return FG_OK;
}

#define PAGED_TRY(expr)               \
  do {                                \
    const int rc_ = (expr);           \
    if (rc_ != FG_OK) return rc_;     \
  } while (0)

extern "C" int fg_paged_append(const fg_paged_cache* c, int layer, float* q_out, const float* q, const float* k,
                               const float* v, int64_t ld, int nHeads, int T, const int32_t* count,
                               const double* cos_tab, const double* sin_tab, int npos, int rot, int half) {
  const char* fn = "fg_paged_append";
  PAGED_TRY(fg::check_paged_cache(c, fn));
  PAGED_TRY(check_step(c, layer, T, fn));
  FG_ARG_CHECK(T == 0 || (k && v), "%s: null argument", fn);
  FG_ARG_CHECK(!q == !q_out, "%s: q and q_out are given together", fn);
  const int nH = q ? nHeads : 0;
  FG_ARG_CHECK(!q || (nHeads > 0 && nHeads <= 1 << 20), "%s: %d query heads", fn, nHeads);
  const int64_t wide = (int64_t)(nH > c->nKvHeads ? nH : c->nKvHeads) * c->dHead;
  FG_ARG_CHECK(ld >= wide, "%s: row stride %lld is below %lld", fn, (long long)ld, (long long)wide);
  FG_ARG_CHECK(q != q_out || !q || ld == (int64_t)nH * c->dHead, "%s: q in place needs rows of %d x %d", fn, nH, c->dHead);
  FG_ARG_CHECK(rot >= 0 && rot <= c->dHead && rot % 2 == 0, "%s: %d rotated values of %d", fn, rot, c->dHead);
  FG_ARG_CHECK(rot == 0 || (cos_tab && sin_tab && npos > 0), "%s: no table of angles", fn);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  const int64_t rows = (int64_t)c->nSeq * T;
  fg::KProfScope prof("paged_append", 0.0, rows * (8.0 * nH * c->dHead + 8.0 * c->nKvHeads * c->dHead + 2 * row_bytes(c)));
  const bool fours = rot % 8 == 0 && ld % 4 == 0 && aligned16(q) && aligned16(q_out) && aligned16(k) && aligned16(v);
#define PAGED_APPEND(KV, P)                                                                                       \
  FG_LAUNCH((paged_append_kernel<KV, P>), dim3((unsigned)rows), dim3(kThreads), 0, view(c), layer, c->dHead, q_out, q, \
            k, v, ld, nH, T, count, cos_tab, sin_tab, npos, rot, half)
  if (c->type == 0) {
    if (fours) PAGED_APPEND(float, 4);
    else PAGED_APPEND(float, 1);
  } else {
    if (fours) PAGED_APPEND(_Float16, 4);
    else PAGED_APPEND(_Float16, 1);
  }
  return FG_OK;
}

extern "C" int fg_paged_read(const fg_paged_cache* c, int layer, float* k, float* v, int64_t ld, int first, int T) {
  const char* fn = "fg_paged_read";
  PAGED_TRY(fg::check_paged_cache(c, fn));
  PAGED_TRY(check_step(c, layer, T, fn));
  FG_ARG_CHECK(first >= 0 && (int64_t)first + T <= (int64_t)c->maxPages * c->pageSize,
               "%s: slots [%d, %lld) outside [0, %lld)", fn, first, (long long)first + T,
               (long long)c->maxPages * c->pageSize);
  FG_ARG_CHECK(T == 0 || (k && v), "%s: null argument", fn);
  FG_ARG_CHECK(ld >= (int64_t)c->nKvHeads * c->dHead, "%s: row stride %lld is below %d x %d", fn, (long long)ld,
               c->nKvHeads, c->dHead);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  const int64_t rows = (int64_t)c->nSeq * T;
  fg::KProfScope prof("paged_read", 0.0, rows * 2 * (4.0 * c->nKvHeads * c->dHead + row_bytes(c)));
  const bool fours = ld % 4 == 0 && aligned16(k) && aligned16(v);
#define PAGED_READ(KV, N)                                                                                            \
  FG_LAUNCH((paged_read_kernel<KV, N>), dim3((unsigned)rows, 2), dim3(kThreads), 0, view(c), layer, c->dHead, k, v, ld, \
            first, T)
  if (c->type == 0) {
    if (fours) PAGED_READ(float, 4);
    else PAGED_READ(float, 1);
  } else {
    if (fours) PAGED_READ(_Float16, 4);
    else PAGED_READ(_Float16, 1);
  }
  return FG_OK;
}

extern "C" int fg_paged_attn(const fg_paged_cache* c, int layer, float* out, const float* q, int nHeads, double scale,
                             int T, const int32_t* count, int window, int sinks) {
  const char* fn = "fg_paged_attn";
  PAGED_TRY(fg::check_paged_cache(c, fn));
  PAGED_TRY(check_step(c, layer, T, fn));
  FG_ARG_CHECK(T == 0 || (out && q), "%s: null argument", fn);
  FG_ARG_CHECK(T == 0 || out != q, "%s: out in place of q", fn);
  FG_ARG_CHECK(nHeads > 0 && nHeads % c->nKvHeads == 0, "%s: %d query heads for %d kv heads", fn, nHeads, c->nKvHeads);
  FG_ARG_CHECK(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", fn, window, sinks);
  const int64_t items = (int64_t)c->nSeq * T * nHeads;
  FG_ARG_CHECK(items <= INT32_MAX / kThreads, "%s: %d sequences x %d tokens x %d heads are too many", fn, c->nSeq, T, nHeads);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("paged_attn", 0.0, (double)c->nSeq * c->maxPages * c->pageSize * 2 * row_bytes(c));
  const int group = nHeads / c->nKvHeads, all = T * group;
  // Many rows share steps through LDS, few take them in registers.  us, shared against registers:
  //   fp16  24 rows of 128, 8 sequences of 8000   64  53     48 rows   76  95     96 rows   86 154
  //         24 rows of 64                        104  48     48 rows  109 122     96 rows  115 189
  //   fp32  64 rows of 128, 8 sequences up to 8000 164 108    96 rows  172 175   128 rows  174 222
  //         64 rows of 64                           94  66    96 rows   96 106   128 rows   98 133
  // (A tile of 64 rows in registers leaves a CU one workgroup: 64 rows of 128 fp32 120, of 64 73.)
  // Heads of 256 leave a wave of 32 rows no registers: 256 rows 116 (two tiles of 16: 65), 1024 rows 261 (152).
  const bool wide = c->dHead < 256 && all > (c->type ? 32 : 64);
  const int tiles = all <= 16 ? 1 : 2;
  const Span span{T, group, wide ? kWideRows : 16 * tiles, window, sinks, (c->type ? 32 : 16) * (wide ? 2 : 1),
                  wide ? 1 : kWaves, count};
  const int64_t heads = (int64_t)c->nSeq * c->nKvHeads * ((all + span.rows - 1) / span.rows);
  const int64_t room = (int64_t)c->maxPages * c->pageSize;
  int64_t seen = room;  // by a workgroup's rows, at most
  if (window > 0 && (int64_t)window + T + sinks + 2 * span.keys < room) seen = (int64_t)window + T + sinks + 2 * span.keys;
  const int64_t rounds = (seen + span.keys * span.waves - 1) / (span.keys * span.waves);
  // Workgroups that the chip holds at once, and, where a workgroup's time is mostly its reads, as many of them as give
  // every head two.
  const int cus = fg::device_cu_count() > 0 ? fg::device_cu_count() : 256;
  const int64_t held = (int64_t)cus * (wide || c->dHead < 256 ? 2 : 1);
  const int64_t target = wide ? held : held * ((2 * heads + held - 1) / held);
  // Short caches, of more slots where there are heads enough to fill the chip: a workgroup a head and tile, no second
  // launch.  A round of it takes about 0.6 us and 0.07 for each KB that a wave reads; pieces and their joining take
  // 6 us more than a round.  us, a workgroup a head against pieces:
  //                        up to the limit              beyond it
  //    8 heads of 128 fp16   512: 12.0 12.0              1024: 19.1 12.1
  //    8 heads of 64 fp16    512:  9.2 11.2              1024: 14.3 11.0
  //    4 heads of 32 fp32    512: 10.3 11.2              1024: 17.5 11.3
  //   48 heads of 64 fp32    256:  8.4 11.2               512: 12.4 12.5
  //    4 heads of 256 fp16   256: 12.1 14.1               512: 18.8 14.3
  //    8 heads, 20 rows      256: 12.4 15.4               512: 17.5 15.5
  //  256 heads of 32 fp32   1024: 23.6 25.3              2048: 42.8 36.6
  //  512 heads of 128 fp16  2048: 95.5 99.5
  const int64_t kb = span.keys * c->dHead * (c->type ? 2 : 4) * 2 / 1024;
  const int64_t limit = (wide ? 2 : tiles > 1 ? 64 / (8 + kb) : 98 / (8 + kb)) * (heads >= cus ? 4 : 1);
  const bool whole = rounds <= (limit > 1 ? limit : 1) || heads >= (wide ? held : 4 * held);
  const int64_t grid = (whole ? heads : heads + target) + 8 * (whole ? (all + span.rows - 1) / span.rows : 1);  // (by_die: a die's run may end beyond the last)
  FG_ARG_CHECK(grid <= INT32_MAX / kThreads, "%s: %d sequences x %d tokens x %d heads are too many", fn, c->nSeq, T, nHeads);
  fg::Workspace ws;
  float2* part_ml = nullptr;
  float* part_o = nullptr;
  Pieces* plan = nullptr;
  int R = 1;
  if (!whole) {
    const size_t rows = (size_t)grid * span.rows;
    PAGED_TRY(ws.get(rows * (sizeof(float2) + c->dHead * sizeof(float)) + c->nSeq * sizeof(Pieces)));
    part_o = (float*)ws.ptr;
    part_ml = (float2*)(part_o + rows * c->dHead);
    plan = (Pieces*)(part_ml + rows);
    while (2 * R <= kThreads / (c->dHead / 4) && items / R > 4 * cus) R *= 2;
  }
  const int64_t joins = (int64_t)c->nSeq * c->nKvHeads * ((all + R - 1) / R);
  const float factor = (float)(scale * M_LOG2E);
  const Cache cache = view(c);
#define PAGED_ATTN(KV, DH, NT)                                                                                        \
  FG_LAUNCH((paged_attn_kernel<KV, DH, NT>), dim3((unsigned)grid), dim3(kThreads), 0, cache, layer, out, q, nHeads,   \
            factor, span, (int)target, plan, part_ml, part_o)
#define PAGED_TILES(KV, DH)                                                                                           \
  if constexpr (DH < 256) {                                                                                           \
    if (wide) {                                                                                                       \
      FG_LAUNCH((paged_wide_kernel<KV, DH>), dim3((unsigned)grid), dim3(kThreads), 0, cache, layer, out, q, nHeads,   \
                factor, span, (int)target, plan, part_ml, part_o);                                                    \
      break;                                                                                                          \
    }                                                                                                                 \
  }                                                                                                                   \
  if (tiles == 1) PAGED_ATTN(KV, DH, 1);                                                                              \
  else PAGED_ATTN(KV, DH, 2)
#define PAGED_HEAD(DH)                               \
  do {                                               \
    do {                                             \
      if (c->type == 0) {                            \
        PAGED_TILES(float, DH);                      \
      } else {                                       \
        PAGED_TILES(_Float16, DH);                   \
      }                                              \
    } while (0);                                     \
    if (!whole)                                      \
      FG_LAUNCH(paged_join_kernel<DH>, dim3((unsigned)joins), dim3(kThreads), 0, cache, out, nHeads, span, R, \
                (const Pieces*)plan, (const float2*)part_ml, (const float*)part_o);                          \
  } while (0)
  switch (c->dHead) {
    case 32: PAGED_HEAD(32); break;
    case 64: PAGED_HEAD(64); break;
    case 96: PAGED_HEAD(96); break;
    case 128: PAGED_HEAD(128); break;
    default: PAGED_HEAD(256); break;
  }
  return FG_OK;
}

extern "C" int fg_paged_commit(const fg_paged_cache* c, int T, const int32_t* count) {
  PAGED_TRY(fg::check_paged_cache(c, "fg_paged_commit"));
  FG_ARG_CHECK(T >= 0, "fg_paged_commit: T %d is negative", T);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("paged_commit", 0.0, 12.0 * c->nSeq);
  FG_LAUNCH(paged_commit_kernel, dim3((c->nSeq + kThreads - 1) / kThreads), dim3(kThreads), 0, view(c), T, count);
  return FG_OK;
}
