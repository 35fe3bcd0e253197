// Verification of drafted tokens (fg_draft_verify): speculative sampling, whose standing
// drafts and the token after them are distributed as the target model's own.
//
// What decides are two numbers of a row, p(x) and q(x) at its draft, but each needs its row's
// sum, so the first launch reads every logit of both models once, in chunks, and leaves a
// greatest logit and a sum of exponentials for each.  The second finds the row that the next
// token is drawn from, a chunk a workgroup, and sums its weights max(p - q, 0); the third finds the
// chunk and in it the token that the given number falls on.
//
// Everything from the exponentials on is fp64: an fp32 sum is off by 1e-7 of itself, which among the
// 1e5 borders between tokens would give another token once in a few thousand draws.  The
// exponentials take about as long as reading the logits does, and mostly beside it.
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 16, kChunk = kThreads * kEach;  // logits of a thread, of a workgroup
constexpr int kLast = 1024;                           // threads of the last launch, 4 logits each
static_assert(kLast * 4 == kChunk, "the last launch takes a chunk");

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
// Logits of chunk c as a thread has them; -inf behind the last.
__device__ __forceinline__ void load_chunk(float (&x)[kEach], const float* row, int c, int V, bool fours) {
  const int from = c * kChunk;
  if (fours && from + kChunk <= V) {
#pragma unroll
    for (int k = 0; k < kEach / 4; ++k) {
      const float4 y = *reinterpret_cast<const float4*>(row + from + (k * kThreads + threadIdx.x) * 4);
      x[4 * k] = y.x, x[4 * k + 1] = y.y, x[4 * k + 2] = y.z, x[4 * k + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int v = from + k * kThreads + threadIdx.x;
      x[k] = v < V ? row[v] : -INFINITY;
    }
  }
}
// Where element k of load_chunk stands.
__device__ __forceinline__ int token_of(int k, int c, int V, bool fours) {
  const int from = c * kChunk;
  return fours && from + kChunk <= V ? from + (k / 4 * kThreads + threadIdx.x) * 4 + k % 4 : from + k * kThreads + threadIdx.x;
}
__device__ __forceinline__ double power(float x, float top, double inv) {
  return x == -INFINITY ? 0.0 : exp(((double)x - (double)top) * inv);
}

// A workgroup takes a chunk of a row: rows of the target model first, then the draft model's.
template <bool Greedy>
__global__ void __launch_bounds__(kThreads) draft_sums_kernel(Sum* __restrict__ sums, Args a, int nSeq) {
  __shared__ float tops[kWaves];
  __shared__ double parts[kWaves];
  __shared__ int ats[kWaves];
  const int64_t row = blockIdx.x / a.chunks;
  const int c = blockIdx.x - (int)row * a.chunks;
  const int64_t targets = (int64_t)nSeq * (a.D + 1);
  const bool second = row >= targets;
  const int s = (int)(second ? (row - targets) / a.D : row / (a.D + 1));
  const int t = (int)(second ? (row - targets) - (int64_t)s * a.D : row - (int64_t)s * (a.D + 1));
  if (t > drafts_of(a, s) - second) return;
  const bool fours = second ? a.draft_fours : a.fours;
  float x[kEach];
  load_chunk(x, second ? draft_row(a, s, t) : target_row(a, s, t), c, a.V, fours);
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
      const int v = token_of(k, c, a.V, fours);
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
    double sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) sum += power(x[k], top, a.inv);
    sum = wave_sum(sum);
    if (lane == 0) parts[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += parts[w];
      sums[blockIdx.x] = Sum{sum, top, 0};
    }
  }
}

// A row's greatest logit and 1 / sum, by a wave.
__device__ __forceinline__ void row_sum(const Sum* sums, const Args& a, float& top, double& back) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, sums[c].top);
  m = fg_wave_max(m);
  double sum = 0;
  for (int c = lane; c < a.chunks; c += 64) {
    const Sum p = sums[c];
    sum += p.sum * power(p.top, m, a.inv);
  }
  sum = wave_sum(sum);
  top = m;
  back = m == -INFINITY ? (double)NAN : 1.0 / sum;
}

// How many drafts of sequence s stand, by the workgroup: a wave a row, kWaves rows at a time.
__device__ Next next_of(const Sum* sums, const Args& a, int s, int nSeq, int n) {
  __shared__ Next rows[kWaves];
  __shared__ int stands[kWaves];
  const int wave = threadIdx.x >> 6;
  for (int t0 = 0;; t0 += kWaves) {
    const int t = t0 + wave;
    if (t <= n) {
      Next r{t, t < n ? a.draft[(int64_t)s * a.D + t] : -1, 0.f, 0.f, 0.0, 0.0};
      row_sum(sums + ((int64_t)s * (a.D + 1) + t) * a.chunks, a, r.ptop, r.pback);
      const bool in = (uint32_t)r.draft < (uint32_t)a.V;
      bool ok = false;
      double q = 1.0;  // of a draft that was certain
      if (t < n && a.draft_logits) {
        row_sum(sums + ((int64_t)nSeq * (a.D + 1) + (int64_t)s * a.D + t) * a.chunks, a, r.qtop, r.qback);
        if (in) q = power(draft_row(a, s, t)[r.draft], r.qtop, a.inv) * r.qback;
      }
      if (t < n && in) ok = (double)a.u[(int64_t)s * (a.D + 1) + t] * q < power(target_row(a, s, t)[r.draft], r.ptop, a.inv) * r.pback;
      if ((threadIdx.x & 63) == 0) {
        rows[wave] = r;
        stands[wave] = ok;
      }
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
      if (!stands[w]) return rows[w];  // at t = n at the latest
    __syncthreads();
  }
}
// max(p - q, 0) of a token, or p where `less` is not set.  Each product is rounded before
// the subtraction: where p and q are equal nothing is left, in every launch.
__device__ __forceinline__ double weight(const Next& r, const Args& a, float x, float y, int v, bool less) {
#pragma clang fp contract(off)
  const double p = power(x, r.ptop, a.inv) * r.pback;
  if (!less) return p;
  const double q = a.draft_logits ? power(y, r.qtop, a.inv) * r.qback : v == r.draft ? 1.0 : 0.0;
  return fmax(p - q, 0.0);
}

// A workgroup takes a chunk of the row that a sequence's next token is drawn from.
__global__ void __launch_bounds__(kThreads) draft_weights_kernel(double* __restrict__ weights, Next* __restrict__ nexts,
                                                                 const Sum* __restrict__ sums, Args a, int nSeq) {
  __shared__ double parts[kWaves];
  const int s = blockIdx.x / a.chunks, c = blockIdx.x - s * a.chunks, n = drafts_of(a, s);
  if (n < 0) return;
  const Next r = next_of(sums, a, s, nSeq, n);
  if (c == 0 && threadIdx.x == 0) nexts[s] = r;
  if (r.taken == n) return;  // no weights but the probabilities
  float x[kEach], y[kEach] = {};
  const bool fours = a.fours && (!a.draft_logits || a.draft_fours);
  load_chunk(x, target_row(a, s, r.taken), c, a.V, fours);
  if (a.draft_logits) load_chunk(y, draft_row(a, s, r.taken), c, a.V, fours);
  double sum = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) sum += weight(r, a, x[k], y[k], token_of(k, c, a.V, fours), true);
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += parts[w];
    weights[blockIdx.x] = sum;
  }
}

__device__ __forceinline__ void write_tokens(int32_t* token, int32_t* count, const Args& a, int s, int taken, int last) {
  for (int t = threadIdx.x; t <= a.D; t += blockDim.x)
    token[(int64_t)s * (a.D + 1) + t] = t < taken ? a.draft[(int64_t)s * a.D + t] : t == taken ? last : -1;
  if (threadIdx.x == 0) count[s] = taken + 1;
}

// A workgroup draws a sequence's next token.
__global__ void __launch_bounds__(kLast) draft_draw_kernel(int32_t* __restrict__ token, int32_t* __restrict__ count,
                                                           const double* __restrict__ weights,
                                                           const Next* __restrict__ nexts, const Sum* __restrict__ sums,
                                                           Args a) {
  constexpr int kLastWaves = kLast / 64;
  __shared__ double parts[kLastWaves];
  __shared__ int found[kLastWaves], ends[kLastWaves];
  __shared__ double start, goal_at;
  __shared__ int chunk_at;
  const int s = blockIdx.x, n = drafts_of(a, s), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (n < 0) {
    write_tokens(token, count, a, s, -1, -1);
    return;
  }
  const Next r = nexts[s];
  const Sum* mine = sums + ((int64_t)s * (a.D + 1) + r.taken) * a.chunks;
  // the chunk: one wave, 64 chunks at a time
  bool less = r.taken < n;
  if (wave == 0) {
    auto chunk_weight = [&](int c) {
      return c >= a.chunks ? 0.0 : less ? weights[(int64_t)s * a.chunks + c] : mine[c].sum * power(mine[c].top, r.ptop, a.inv) * r.pback;
    };
    double all = 0;
    for (;; less = false) {
      all = 0;
      for (int c = lane; c < a.chunks; c += 64) all += chunk_weight(c);
      all = wave_sum(all);
      if (all > 0 || !less) break;
    }
    const double goal = (double)a.u[(int64_t)s * (a.D + 1) + a.D] * all;
    int at = -1;
    double before = 0, run = 0;
    if (all > 0 && r.pback == r.pback) {
      for (int c0 = 0; c0 < a.chunks; c0 += 64) {
        const double w = chunk_weight(c0 + lane);
        double upto = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double below = __shfl_up(upto, o, 64);
          if (lane >= o) upto += below;
        }
        upto += run;
        const uint64_t some = __ballot(w > 0), over = __ballot(w > 0 && upto > goal);
        const int who = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        if (who >= 0) {
          at = c0 + who;
          before = __shfl(upto - w, who, 64);
        }
        run = __shfl(upto, 63, 64);
        if (over) break;
      }
    }
    if (lane == 0) {
      chunk_at = at;
      start = before;
      goal_at = goal;
      ends[0] = less;
    }
  }
  __syncthreads();
  const int c = chunk_at;
  less = ends[0] != 0;
  const double goal = goal_at;
  if (c < 0) {
    write_tokens(token, count, a, s, r.taken, -1);
    return;
  }
  // the token: four neighbours a thread
  const int v0 = c * kChunk + threadIdx.x * 4;
  const float *x = target_row(a, s, r.taken), *y = less && a.draft_logits ? draft_row(a, s, r.taken) : nullptr;
  double w[4], sum = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int v = v0 + k;
    w[k] = v < a.V ? weight(r, a, x[v], y ? y[v] : 0.f, v, less) : 0.0;
    sum += w[k];
  }
  double upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double below = __shfl_up(upto, o, 64);
    if (lane >= o) upto += below;
  }
  if (lane == 63) parts[wave] = upto;
  __syncthreads();
  double reach = start;
  for (int v = 0; v < wave; ++v) reach += parts[v];
  reach += upto - sum;
  int at = INT32_MAX, end = -1;  // the token, and the last of any weight
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    reach += w[k];
    if (w[k] > 0) {
      end = v0 + k;
      if (reach > goal) at = min(at, v0 + k);
    }
  }
  at = wave_min(at);
  end = -wave_min(-end);
  __syncthreads();
  if (lane == 0) {
    found[wave] = at;
    ends[wave] = end;
  }
  __syncthreads();
  at = INT32_MAX, end = -1;
  for (int v = 0; v < kLastWaves; ++v) {
    at = min(at, found[v]);
    end = max(end, ends[v]);
  }
  write_tokens(token, count, a, s, r.taken, at != INT32_MAX ? at : end);
}

// Temperature 0: a workgroup takes a sequence, a wave a row.
__global__ void __launch_bounds__(kThreads) draft_greedy_kernel(int32_t* __restrict__ token, int32_t* __restrict__ count,
                                                                const Sum* __restrict__ sums, Args a) {
  __shared__ int best[kWaves];
  const int s = blockIdx.x, n = drafts_of(a, s), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (n < 0) {
    write_tokens(token, count, a, s, -1, -1);
    return;
  }
  for (int t0 = 0;; t0 += kWaves) {
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
    for (int w = 0; w < kWaves; ++w) {
      const int b = best[w];
      if (t0 + w == n || b < 0 || a.draft[(int64_t)s * a.D + t0 + w] != b) {
        write_tokens(token, count, a, s, t0 + w, b);
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
  const size_t sums_bytes = (size_t)rows * chunks * sizeof(Sum), next_bytes = (size_t)nSeq * sizeof(Next);
  const size_t weight_bytes = (size_t)nSeq * chunks * sizeof(double);
  fg::Workspace ws;
  const int rc = ws.get(sums_bytes + next_bytes + weight_bytes);
  if (rc != FG_OK) return rc;
  Sum* sums = (Sum*)ws.ptr;
  double* weights = (double*)((uint8_t*)ws.ptr + sums_bytes);
  Next* nexts = (Next*)((uint8_t*)ws.ptr + sums_bytes + weight_bytes);
  const dim3 all((unsigned)(rows * chunks)), row((unsigned)(nSeq * chunks)), seq((unsigned)nSeq);
  if (temperature == 0) {
    FG_LAUNCH(draft_sums_kernel<true>, all, dim3(kThreads), 0, sums, a, nSeq);
    FG_LAUNCH(draft_greedy_kernel, seq, dim3(kThreads), 0, token, count, (const Sum*)sums, a);
    return FG_OK;
  }
  FG_LAUNCH(draft_sums_kernel<false>, all, dim3(kThreads), 0, sums, a, nSeq);
  FG_LAUNCH(draft_weights_kernel, row, dim3(kThreads), 0, weights, nexts, (const Sum*)sums, a, nSeq);
  FG_LAUNCH(draft_draw_kernel, seq, dim3(kLast), 0, token, count, (const double*)weights, (const Next*)nexts,
            (const Sum*)sums, a);
  return FG_OK;
}
