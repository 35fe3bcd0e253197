// Verification of drafted tokens (fg_draft_verify): speculative sampling, whose standing
// drafts and the token after them are distributed as the target model's own.
//
// What decides are two numbers of a row, p(x) and q(x) at its draft, but each needs its row's
// sum, so the first launch reads every logit of both models once, in chunks, and leaves a
// greatest logit and a sum of exponentials for each.  The second finds the row that the next
// token is drawn from and sums its weights max(p - q, 0), a piece a wave; the third finds the
// piece, and in it the token, that the given number falls on (the second does where a workgroup has the
// whole row.  Letting the last of a sequence's workgroups draw, instead of a launch, needs their sums to be
// written back between the dies' caches first: 48 us against 12 and 8).
//
// Probabilities, sums and comparisons are fp64: an fp32 sum is off by 1e-7 of itself, which among the
// 1e5 borders between tokens would give another token once in a few thousand draws.  The sums' exponentials are good
// to 2.2e-10 (Quick).
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 16, kChunk = kThreads * kEach;  // logits of a thread, of a workgroup of the first launch
constexpr int kDrawWaves = 16;               // of a workgroup of the launches that draw

__device__ __forceinline__ double wave_sum(double x) { return fg_wave_sum_d(x); }
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
  return x;
}

struct Args {
  const float *logits, *draft_logits;
  int64_t ld, ld_draft;
  const int32_t *draft, *drafted;
  const float* u;
  double inv;  // 1 / temperature
  int D, V, chunks;
  bool fours, draft_fours;  // rows are aligned to 16 bytes
};
// A chunk's greatest logit and sum of exp((x - top) inv); greedy: its lowest token in `at`.
struct alignas(16) Sum {
  double sum;
  float top;
  int at;
};
// The row that the next token of a sequence is drawn from.
struct Next {
  int taken, draft;     // drafts that stand, the next one (-1: none)
  float ptop, qtop;
  double pback, qback;  // 1 / sums; q is 0 everywhere where qback is 0
};

__device__ __forceinline__ int drafts_of(const Args& a, int s) { return a.drafted ? min(a.drafted[s], a.D) : a.D; }
__device__ __forceinline__ const float* target_row(const Args& a, int s, int t) {
  return a.logits + ((int64_t)s * (a.D + 1) + t) * a.ld;
}
__device__ __forceinline__ const float* draft_row(const Args& a, int s, int t) {
  return a.draft_logits + ((int64_t)s * a.D + t) * a.ld_draft;
}
// N logits a thread from `from` on, a wave's neighbours; -inf behind the last.  Runs of four where rows are aligned.
template <int N>
__device__ __forceinline__ void load_logits(float (&x)[N], const float* row, int from, int V, bool fours) {
  const int lane = threadIdx.x & 63;
  if (fours && from + 64 * N <= V) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const float4 y = *reinterpret_cast<const float4*>(row + from + (k * 64 + lane) * 4);
      x[4 * k] = y.x, x[4 * k + 1] = y.y, x[4 * k + 2] = y.z, x[4 * k + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = from + k * 64 + lane;
      x[k] = v < V ? row[v] : -INFINITY;
    }
  }
}
// Where element k of load_logits stands.
template <int N>
__device__ __forceinline__ int token_of(int k, int from, int V, bool fours) {
  const int lane = threadIdx.x & 63;
  return fours && from + 64 * N <= V ? from + (k / 4 * 64 + lane) * 4 + k % 4 : from + k * 64 + lane;
}
__device__ __forceinline__ double power(float x, float top, double inv) {
  return x == -INFINITY ? 0.0 : exp(((double)x - (double)top) * inv);
}

// exp((x - top) inv) for the sums: t = (x - top) inv log2 e in 1/256ths, its whole part from a table of 256 and the
// exponent, the rest, up to 1/512, by a polynomial whose roundings are fp32's, of something below 1.4e-3: 2.2e-10 of the
// exponential at most, 4e-11 as a deviation, of both signs.  They cancel where terms differ (1e-12 of a sum of a thousand such), and do
// not where they are equal; a number as near to a border may fall on its other side.
// 19 instructions; exp takes 30, and 16 sequences of 9 rows of
// 128256 logits then 18 us instead of 27 (13 with fp32 exponentials).
constexpr int kSteps = 256;
struct Quick {
  const double* table;  // 2^(j / kSteps), LDS
  double top, k;
  __device__ __forceinline__ double at(float x) const {
    // below 2^-1000 all the same; NaN is the caller's
    const double t = fmax(((double)x - top) * k, -1000.0 * kSteps), whole = t + 0x1.8p52;
    const int n = __double2loint(whole);
    const float f = (float)(t - (whole - 0x1.8p52)) * (float)(M_LN2 / kSteps);
    const float c = f * fmaf(f, fmaf(f, 1.f / 6, 0.5f), 1.f);
    const double base = table[n & (kSteps - 1)], y = fma(base, (double)c, base);
    return __hiloint2double(__double2hiint(y) + (n >> 8 << 20), __double2loint(y));
  }
};

// A workgroup takes a chunk of a row: rows of the target model first, then the draft model's.
template <bool Greedy>
__global__ void __launch_bounds__(kThreads) draft_sums_kernel(Sum* __restrict__ sums, Args a, int nSeq) {
  __shared__ float tops[kWaves];
  __shared__ double parts[kWaves], table[kSteps];
  __shared__ int ats[kWaves];
  static_assert(kSteps == kThreads, "a thread an entry");
  const int64_t row = blockIdx.x / a.chunks;
  const int c = blockIdx.x - (int)row * a.chunks;
  const int64_t targets = (int64_t)nSeq * (a.D + 1);
  const bool second = row >= targets;
  const int s = (int)(second ? (row - targets) / a.D : row / (a.D + 1));
  const int t = (int)(second ? (row - targets) - (int64_t)s * a.D : row - (int64_t)s * (a.D + 1));
  if (t > drafts_of(a, s) - second) return;
  const bool fours = second ? a.draft_fours : a.fours;
  float x[kEach];
  const int from = c * kChunk + (int)(threadIdx.x >> 6) * (64 * kEach);
  load_logits(x, second ? draft_row(a, s, t) : target_row(a, s, t), from, a.V, fours);
  if constexpr (!Greedy) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / kSteps));
  float top = x[0];
#pragma unroll
  for (int k = 1; k < kEach; ++k) top = fmaxf(top, x[k]);
  top = fg_wave_max(top);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = tops[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, tops[w]);
  if constexpr (Greedy) {
    int at = INT32_MAX;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int v = token_of<kEach>(k, from, a.V, fours);
      if (x[k] == top && v < a.V) at = min(at, v);
    }
    at = wave_min(at);
    if (lane == 0) ats[wave] = at;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) at = min(at, ats[w]);
      sums[blockIdx.x] = Sum{0.0, top, at};
    }
  } else {
    bool number = top < INFINITY;  // all of them below infinity
#pragma unroll
    for (int k = 0; k < kEach; ++k) number &= x[k] == x[k];
    double sum = 0;
    if (top > -INFINITY) {
      const Quick quick{table, top, a.inv * (M_LOG2E * kSteps)};
#pragma unroll
      for (int k = 0; k < kEach; ++k) sum += quick.at(x[k]);
    }
    sum = wave_sum(number ? sum : (double)NAN);
    if (lane == 0) parts[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += parts[w];
      sums[blockIdx.x] = Sum{sum, top, 0};
    }
  }
}

// A lane's share of a row's chunks, its own numbers asked for at once where there are up to 64, and, of a wave's
// lanes, the row's greatest logit and 1 / sum.
__device__ __forceinline__ Sum lanes_chunk(const Sum* sums, const Args& a) {
  const int lane = threadIdx.x & 63;
  return lane < a.chunks ? sums[lane] : Sum{0.0, -INFINITY, 0};
}
__device__ __forceinline__ void row_sum(Sum p, const Sum* sums, const Args& a, float& top, double& back) {
  for (int c = (threadIdx.x & 63) + 64; c < a.chunks; c += 64) {
    const Sum z = sums[c];
    const float m = fmaxf(p.top, z.top);
    p.sum = p.sum * power(p.top, m, a.inv) + z.sum * power(z.top, m, a.inv);
    p.top = m;
  }
  const float m = fg_wave_max(p.top);
  const double sum = wave_sum(p.sum * power(p.top, m, a.inv));
  top = m;
  back = m == -INFINITY ? (double)NAN : 1.0 / sum;
}

// How many drafts of sequence s stand, by the workgroup: a wave a row, kDrawWaves rows at a time.
__device__ Next next_of(const Sum* sums, const Args& a, int s, int nSeq, int n) {
  __shared__ Next rows[kDrawWaves];
  __shared__ int stands[kDrawWaves];
  const int wave = threadIdx.x >> 6;
  for (int t0 = 0;; t0 += kDrawWaves) {
    const int t = t0 + wave;
    if (t <= n) {
      const bool two = t < n && a.draft_logits;
      const Sum* const ps = sums + ((int64_t)s * (a.D + 1) + t) * a.chunks;
      const Sum* const qs = sums + ((int64_t)nSeq * (a.D + 1) + (int64_t)s * a.D + t) * a.chunks;
      // (the draft first, whose logits are asked for when it is there, before the sums are waited for)
      Next r{t, t < n ? a.draft[(int64_t)s * a.D + t] : -1, 0.f, 0.f, 0.0, 0.0};
      const float u = t < n ? a.u[(int64_t)s * (a.D + 1) + t] : 0.f;
      const Sum p = lanes_chunk(ps, a), q = two ? lanes_chunk(qs, a) : Sum{};
      const bool in = t < n && (uint32_t)r.draft < (uint32_t)a.V;
      const float x = in ? target_row(a, s, t)[r.draft] : 0.f, y = in && two ? draft_row(a, s, t)[r.draft] : 0.f;
      row_sum(p, ps, a, r.ptop, r.pback);
      if (two) row_sum(q, qs, a, r.qtop, r.qback);
      const double share = two ? power(y, r.qtop, a.inv) * r.qback : 1.0;  // 1: of a draft that was certain
      const bool ok = in && (double)u * share < power(x, r.ptop, a.inv) * r.pback;
      if ((threadIdx.x & 63) == 0) {
        rows[wave] = r;
        stands[wave] = ok;
      }
    }
    __syncthreads();
    for (int w = 0; w < kDrawWaves; ++w)
      if (!stands[w]) return rows[w];  // at t = n at the latest
    __syncthreads();
  }
}
// p of a token, and max(p - q, 0) where `less` is set.  Each product is rounded before
// the subtraction: where p and q are equal nothing is left, wherever this is computed.
__device__ __forceinline__ double weight(const Next& r, const Args& a, float x, float y, int v, bool less, double& p) {
#pragma clang fp contract(off)
  p = power(x, r.ptop, a.inv) * r.pback;
  if (!less) return p;
  const double q = a.draft_logits ? power(y, r.qtop, a.inv) * r.qback : v == r.draft ? 1.0 : 0.0;
  return fmax(p - q, 0.0);
}

// Thread t's draft (up to 1023 drafts, a thread each), asked for before it is known whether it stands.
static_assert(64 * kDrawWaves >= 1024, "a thread a draft");
__device__ __forceinline__ int own_draft(const Args& a, int s) {
  return (int)threadIdx.x < a.D ? a.draft[(int64_t)s * a.D + threadIdx.x] : -1;
}
__device__ __forceinline__ void write_tokens(int32_t* token, int32_t* count, const Args& a, int s, int taken, int last, int own) {
  const int t = threadIdx.x;
  if (t <= a.D) token[(int64_t)s * (a.D + 1) + t] = t < taken ? own : t == taken ? last : -1;
  if (t == 0) count[s] = taken + 1;
}

// The inclusive sums of 64 lanes' x.
__device__ __forceinline__ double lanes_upto(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double below = __shfl_up(x, o, 64);
    if ((int)(threadIdx.x & 63) >= o) x += below;
  }
  return x;
}

// The token of a sequence's row r that its number falls on, by the workgroup; weights[piece]: the
// weights' sums (both kinds, max(p - q, 0) and p, where drafts are left).  Weights of 2^-40 in all at most are
// what roundings leave of equal rows, summed in other orders.
template <int E>
__device__ int draw(const double* weights, const Next& r, const Args& a, int s, bool less, float u) {
  __shared__ double parts[E], shared_start, shared_goal;  // E waves take a piece
  __shared__ int found[E], ends[E], shared_at, shared_less;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pieces = (a.V + (64 * E) - 1) / (64 * E);
  if (wave == 0) {  // the piece: neighbours a lane
    const int each = (pieces + 63) / 64, from = min(lane * each, pieces), to = min(from + each, pieces);
    double mine, upto, all;
    for (;; less = false) {
      mine = 0;
      for (int z = from; z < to; ++z) mine += weights[2 * z + !less];
      upto = lanes_upto(mine);
      all = __shfl(upto, 63, 64);
      if (all > 0x1p-40 || !less) break;
    }
    const double goal = (double)u * all;
    const uint64_t some = __ballot(mine > 0), over = __ballot(mine > 0 && upto > goal);
    const int who = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
    if (lane == (all > 0 ? who : 0)) {
      int at = -1;
      double reach = upto - mine, before = 0;
      if (all > 0)
        for (int z = from; z < to; ++z) {
          const double w = weights[2 * z + !less];
          if (w > 0) at = z, before = reach;  // the last of any weight where none reaches the goal
          reach += w;
          if (w > 0 && reach > goal) break;
        }
      shared_at = at;
      shared_start = before;
      shared_goal = goal;
      shared_less = less;
    }
  }
  __syncthreads();
  if (shared_at < 0) return -1;
  less = shared_less != 0;
  // the token: one a thread, of the first waves
  const int v = shared_at * (64 * E) + threadIdx.x;
  const bool in = threadIdx.x < (64 * E) && v < a.V;
  double p, w = 0;
  if (in) w = weight(r, a, target_row(a, s, r.taken)[v], less && a.draft_logits ? draft_row(a, s, r.taken)[v] : 0.f, v, less, p);
  const double upto = lanes_upto(w);
  if (lane == 63 && wave < E) parts[wave] = upto;
  __syncthreads();
  double reach = shared_start;
#pragma unroll
  for (int z = 0; z < E; ++z) reach += z < wave ? parts[z] : 0.0;
  reach += upto;
  const uint64_t some = __ballot(w > 0), over = __ballot(w > 0 && reach > shared_goal);
  if (lane == 0 && wave < E) {
    found[wave] = over ? v + __builtin_ctzll(over) : INT32_MAX;
    ends[wave] = some ? v + 63 - __builtin_clzll(some) : -1;
  }
  __syncthreads();
  int at = INT32_MAX, end = -1;  // the token, and the last of any weight
#pragma unroll
  for (int z = 0; z < E; ++z) {
    at = min(at, found[z]);
    end = max(end, ends[z]);
  }
  return at != INT32_MAX ? at : end;
}

// A workgroup takes pieces of the row that a sequence's next token is drawn from, a wave one of 64 E logits.
// Alone: it has all of them, and draws.
template <int E, bool Alone>
__global__ void __launch_bounds__(64 * kDrawWaves) draft_weights_kernel(int32_t* __restrict__ token,
                                                                        int32_t* __restrict__ count, double* weights,
                                                                        Next* __restrict__ nexts,
                                                                        const Sum* __restrict__ sums, Args a, int nSeq,
                                                                        int groups) {
  const int s = blockIdx.x / groups, c = blockIdx.x - s * groups, n = drafts_of(a, s);
  if (n < 0) {
    if (Alone) write_tokens(token, count, a, s, -1, -1, -1);
    return;
  }
  const int own = Alone ? own_draft(a, s) : -1;
  const float u = Alone ? a.u[(int64_t)s * (a.D + 1) + a.D] : 0.f;
  const Next r = next_of(sums, a, s, nSeq, n);
  const bool less = r.taken < n;  // else there are no weights but the probabilities
  float x[E], y[E] = {};
  const bool two = less && a.draft_logits, fours = a.fours && (!two || a.draft_fours);
  const int piece = c * kDrawWaves + (threadIdx.x >> 6), pieces = (a.V + (64 * E) - 1) / (64 * E);
  if (piece >= pieces && !Alone) return;
  load_logits(x, target_row(a, s, r.taken), piece * (64 * E), a.V, fours);
  if (two) load_logits(y, draft_row(a, s, r.taken), piece * (64 * E), a.V, fours);
  double sum = 0, whole = 0;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    double p;
    sum += weight(r, a, x[k], y[k], token_of<E>(k, piece * (64 * E), a.V, fours), less, p);
    whole += p;
  }
  sum = wave_sum(sum);
  whole = wave_sum(whole);
  __shared__ double here[2 * kDrawWaves];
  double* const mine = Alone ? here : weights + (int64_t)s * 2 * pieces;
  if ((threadIdx.x & 63) == 0 && piece < pieces) {
    mine[2 * piece] = sum;
    mine[2 * piece + 1] = whole;
  }
  if constexpr (Alone) {
    __syncthreads();
    write_tokens(token, count, a, s, r.taken, draw<E>(here, r, a, s, less, u), own);
  } else {
    if (c == 0 && threadIdx.x == 0) nexts[s] = r;
  }
}
// A workgroup draws a sequence's next token.
template <int E>
__global__ void __launch_bounds__(64 * kDrawWaves) draft_draw_kernel(int32_t* __restrict__ token,
                                                                     int32_t* __restrict__ count,
                                                                     const double* __restrict__ weights,
                                                                     const Next* __restrict__ nexts, Args a) {
  const int s = blockIdx.x, n = drafts_of(a, s), pieces = (a.V + (64 * E) - 1) / (64 * E);
  if (n < 0) {
    write_tokens(token, count, a, s, -1, -1, -1);
    return;
  }
  const int own = own_draft(a, s);
  const float u = a.u[(int64_t)s * (a.D + 1) + a.D];
  const Next r = nexts[s];
  write_tokens(token, count, a, s, r.taken, draw<E>(weights + (int64_t)s * 2 * pieces, r, a, s, r.taken < n, u), own);
}

// Temperature 0: a workgroup takes a sequence, a wave a row.
__global__ void __launch_bounds__(64 * kDrawWaves) draft_greedy_kernel(int32_t* __restrict__ token,
                                                                       int32_t* __restrict__ count,
                                                                       const Sum* __restrict__ sums, Args a) {
  __shared__ int best[kDrawWaves];
  const int s = blockIdx.x, n = drafts_of(a, s), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (n < 0) {
    write_tokens(token, count, a, s, -1, -1, -1);
    return;
  }
  const int own = own_draft(a, s);
  for (int t0 = 0;; t0 += kDrawWaves) {
    const int t = t0 + wave;
    if (t <= n) {
      const Sum* mine = sums + ((int64_t)s * (a.D + 1) + t) * a.chunks;
      float m = -INFINITY;
      for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, mine[c].top);
      m = fg_wave_max(m);
      int at = INT32_MAX;
      for (int c = lane; c < a.chunks; c += 64)
        if (mine[c].top == m) at = min(at, mine[c].at);
      at = wave_min(at);
      if (lane == 0) best[wave] = at == INT32_MAX ? -1 : at;
    }
    __syncthreads();
    for (int w = 0; w < kDrawWaves; ++w) {
      const int b = best[w];
      if (t0 + w == n || b < 0 || a.draft[(int64_t)s * a.D + t0 + w] != b) {
        write_tokens(token, count, a, s, t0 + w, b, own);
        return;
      }
    }
    __syncthreads();
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int fg_draft_verify(int32_t* token, int32_t* count, const float* logits, int64_t ld,
                               const float* draft_logits, int64_t ld_draft, const int32_t* draft,
                               const int32_t* drafted, const float* u, double temperature, int nSeq, int D, int V) {
  const char* fn = "fg_draft_verify";
  FG_ARG_CHECK(nSeq > 0 && D >= 0 && D <= 1023 && V > 0 && V <= 1 << 26 && (int64_t)nSeq * (D + 1) <= 65535 * 16,
               "%s: bad dimensions: %d sequences of %d drafts, %d tokens", fn, nSeq, D, V);
  FG_ARG_CHECK(temperature == 0 || (temperature >= 1e-30 && temperature < INFINITY), "%s: temperature %g", fn, temperature);
  FG_ARG_CHECK(token && count && logits && (D == 0 || draft) && (temperature == 0 || u), "%s: null argument", fn);
  FG_ARG_CHECK(ld >= V, "%s: row stride %lld is below %d", fn, (long long)ld, V);
  const bool drawn = draft_logits && D > 0 && temperature > 0;
  FG_ARG_CHECK(!drawn || ld_draft >= V, "%s: the drafts' row stride %lld is below %d", fn, (long long)ld_draft, V);
  const int chunks = (V + kChunk - 1) / kChunk;
  const int64_t rows = (int64_t)nSeq * (D + 1 + (drawn ? D : 0));
  FG_ARG_CHECK(rows * chunks <= INT32_MAX / kThreads, "%s: %d sequences of %d drafts over %d tokens are too many", fn,
               nSeq, D, V);
  FG_REQUIRE_INIT();
  fg::KProfScope prof("draft_verify", 0.0, 4.0 * V * rows);
  const Args a{logits, drawn ? draft_logits : nullptr, ld, ld_draft, draft, drafted, u, temperature == 0 ? 0.0 : 1.0 / temperature,
               D, V, chunks, ld % 4 == 0 && aligned16(logits), drawn && ld_draft % 4 == 0 && aligned16(draft_logits)};
  // Logits of a thread of the second launch.  Few, where there are workgroups for all of them at once: each first finds
  // the row that is drawn from, 5 us, and 16 logits take 5 more (7 rows of 32000: 4 a thread 6.8 us, 16 11.9; 16 rows of
  // 128256: 4 a thread, two rounds of workgroups, 15 us, 8 12).
  const int cus = fg::device_cu_count() > 0 ? fg::device_cu_count() : 256;
  auto groups_of = [&](int each) { return (V + 64 * kDrawWaves * each - 1) / (64 * kDrawWaves * each); };
  const int each = (int64_t)nSeq * groups_of(4) <= cus ? 4 : (int64_t)nSeq * groups_of(8) <= cus ? 8 : 16;
  const int groups = groups_of(each), pieces = (V + 64 * each - 1) / (64 * each);
  const size_t sums_bytes = (size_t)rows * chunks * sizeof(Sum), next_bytes = (size_t)nSeq * sizeof(Next);
  const size_t weight_bytes = (size_t)nSeq * 2 * pieces * sizeof(double);
  fg::Workspace ws;
  const int rc = ws.get(sums_bytes + next_bytes + weight_bytes);
  if (rc != FG_OK) return rc;
  Sum* sums = (Sum*)ws.ptr;
  double* weights = (double*)((uint8_t*)ws.ptr + sums_bytes);
  Next* nexts = (Next*)((uint8_t*)ws.ptr + sums_bytes + weight_bytes);
  const dim3 all((unsigned)(rows * chunks)), row((unsigned)(nSeq * groups)), block(64 * kDrawWaves);
  if (temperature == 0) {
    FG_LAUNCH(draft_sums_kernel<true>, all, dim3(kThreads), 0, sums, a, nSeq);
    FG_LAUNCH(draft_greedy_kernel, dim3(nSeq), block, 0, token, count, (const Sum*)sums, a);
    return FG_OK;
  }
  FG_LAUNCH(draft_sums_kernel<false>, all, dim3(kThreads), 0, sums, a, nSeq);
#define DRAFT_DRAW(E)                                                                                                  \
  do {                                                                                                                 \
    if (groups == 1) {                                                                                                 \
      FG_LAUNCH((draft_weights_kernel<E, true>), row, block, 0, token, count, weights, nexts, (const Sum*)sums, a,     \
                nSeq, groups);                                                                                         \
    } else {                                                                                                           \
      FG_LAUNCH((draft_weights_kernel<E, false>), row, block, 0, token, count, weights, nexts, (const Sum*)sums, a,    \
                nSeq, groups);                                                                                         \
      FG_LAUNCH(draft_draw_kernel<E>, dim3(nSeq), block, 0, token, count, (const double*)weights, (const Next*)nexts, a); \
    }                                                                                                                  \
  } while (0)
  if (each == 4) DRAFT_DRAW(4);
  else if (each == 8) DRAFT_DRAW(8);
  else DRAFT_DRAW(16);
  return FG_OK;
}
