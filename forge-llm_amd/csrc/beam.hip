// Beam search (fg_beam_*): the choice of the next beams over beams and
// vocabulary, and the beams' states following their parents in place.
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBeams = 64;

// ── selection ─────────────────────────────────────────────────────────────
// Whether (x, i) comes before (y, j): the greater value, NaN last, then the
// lower index.
template <typename F>
__device__ __forceinline__ bool before(F x, int i, F y, int j) {
  if (x > y) return true;
  if (x < y) return false;
  const bool nx = x != x, ny = y != y;
  if (nx != ny) return ny;
  return i < j;
}

constexpr int kNone = 0x7FFFFFFF;  // index of no candidate, after all others
// The first of the workgroup's (x, i).
__device__ __forceinline__ void block_first(float& x, int& i, float* shx, int* shi) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float y = __shfl_xor(x, o, 64);
    const int j = __shfl_xor(i, o, 64);
    if (i == kNone || (j != kNone && before(y, j, x, i))) x = y, i = j;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shx[threadIdx.x >> 6] = x, shi[threadIdx.x >> 6] = i;
  __syncthreads();
  x = shx[0], i = shi[0];
  for (int w = 1; w < kWaves; ++w)
    if (i == kNone || (shi[w] != kNone && before(shx[w], shi[w], x, i))) x = shx[w], i = shi[w];
}

// One workgroup per beam: log sum exp of its logits, then its W first
// candidates one after the other, into val / tok [beam][W].
__global__ void __launch_bounds__(kThreads) beam_row_kernel(double* __restrict__ val, int32_t* __restrict__ tok,
                                                            const float* __restrict__ logits, int64_t ld,
                                                            const float* __restrict__ scores,
                                                            const int32_t* __restrict__ done, int eos, int W, int V) {
  __shared__ float shx[kWaves];
  __shared__ int shi[kWaves];
  __shared__ double shd[kWaves];
  const int64_t b = blockIdx.x;
  const float* x = logits + b * ld;
  val += b * W;
  tok += b * W;
  if (done && done[b]) {
    if (threadIdx.x < W) {
      val[threadIdx.x] = scores[b];
      tok[threadIdx.x] = threadIdx.x == 0 ? eos : kNone;
    }
    return;
  }
  float m = -INFINITY;
  int at = kNone, nan = 0;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    if (at == kNone || before(x[j], j, m, at)) m = x[j], at = j;
    nan |= x[j] != x[j];
  }
  block_first(m, at, shx, shi);
  nan = __syncthreads_or(nan);
  double sum = 0.0;
  for (int j = threadIdx.x; j < V; j += kThreads) sum += exp((double)x[j] - (double)m);
  sum = fg_wave_sum_d(sum);
  if ((threadIdx.x & 63) == 0) shd[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kWaves; ++w) sum += shd[w];
  double base = (double)scores[b] - ((double)m + log(sum));
  if (nan || m == INFINITY) base = NAN;
  else if (m == -INFINITY) base = -INFINITY;
  const bool flat = !(fabs(base) < INFINITY);  // all candidates are `base`
  float px = 0.f;
  int pi = -1;
  for (int w = 0; w < W; ++w) {
    float bx = 0.f;
    int bi = kNone;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float y = flat ? 0.f : x[j];
      if (pi >= 0 && !before(px, pi, y, j)) continue;
      if (bi == kNone || before(y, j, bx, bi)) bx = y, bi = j;
    }
    block_first(bx, bi, shx, shi);
    if (threadIdx.x == 0) {
      val[w] = flat ? base : base + (double)bx;
      tok[w] = bi;
    }
    if (bi == kNone) {
      for (int i = w + 1 + threadIdx.x; i < W; i += kThreads) tok[i] = kNone;
      return;
    }
    px = bx, pi = bi;
  }
}

// One wave per request, a lane per beam: the greatest head of the beams' sorted
// lists, W times.
__global__ void __launch_bounds__(64) beam_merge_kernel(float* __restrict__ score_out, int32_t* __restrict__ token,
                                                        int32_t* __restrict__ parent, int32_t* __restrict__ done_out,
                                                        const double* __restrict__ val, const int32_t* __restrict__ tok,
                                                        const int32_t* __restrict__ done, int eos, int W) {
  const int lane = threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.x * W;
  const bool on = lane < W;
  const double* vs = val + (r0 + lane) * W;
  const int32_t* ts = tok + (r0 + lane) * W;
  const int fin = on && done ? done[r0 + lane] != 0 : 0;
  int at = 0, mine = on ? ts[0] : kNone;
  double v = on ? vs[0] : 0.0;
  for (int w = 0; w < W; ++w) {
    double best = v;
    int beam = mine == kNone ? kNone : lane;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double y = __shfl_xor(best, o, 64);
      const int j = __shfl_xor(beam, o, 64);
      if (beam == kNone || (j != kNone && before(y, j, best, beam))) best = y, beam = j;
    }
    if (beam == lane) {
      score_out[r0 + w] = (float)v;
      token[r0 + w] = mine;
      parent[r0 + w] = lane;
      if (done_out) done_out[r0 + w] = fin || mine == eos;
      ++at;
      mine = at < W ? ts[at] : kNone;
      v = at < W ? vs[at] : 0.0;
    }
  }
}

// ── states ────────────────────────────────────────────────────────────────
// A thread holds one place of a part, `U` bytes of it, in every beam of the
// request: it reads what the beams take, then writes, so no second buffer and
// no order between threads is needed.
template <typename U, int WM>
__global__ void __launch_bounds__(kThreads) beam_reorder_kernel(uint8_t* __restrict__ base, int64_t beam_stride,
                                                                int64_t outer_stride, int inner, int64_t inner_stride,
                                                                int64_t row_bytes, int rows,
                                                                const int32_t* __restrict__ parent,
                                                                const int32_t* __restrict__ len, int W) {
  __shared__ int from[WM];
  __shared__ int64_t end[WM];
  const int64_t r0 = (int64_t)blockIdx.z * W;
  if (threadIdx.x < WM) {
    int p = threadIdx.x;
    int64_t e = 0;
    if (p < W) {
      const int q = parent[r0 + p];
      if (q >= 0 && q < W && q != p) {
        p = q;
        e = (len ? min(max(len[r0 + p], 0), rows) : rows) * row_bytes;
      }
    }
    from[threadIdx.x] = p;
    end[threadIdx.x] = e;
  }
  __syncthreads();
  uint8_t* part = base + r0 * beam_stride + (blockIdx.y / inner) * outer_stride + (blockIdx.y % inner) * inner_stride;
  int64_t most = 0;
  for (int b = 0; b < W; ++b) most = end[b] > most ? end[b] : most;
  for (int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * sizeof(U); at < most;
       at += (int64_t)gridDim.x * kThreads * sizeof(U)) {
    U v[WM];
#pragma unroll
    for (int b = 0; b < WM; ++b)
      if (at < end[b]) v[b] = *reinterpret_cast<const U*>(part + from[b] * beam_stride + at);
#pragma unroll
    for (int b = 0; b < WM; ++b)
      if (at < end[b]) *reinterpret_cast<U*>(part + b * beam_stride + at) = v[b];
  }
}

template <typename U>
int launch_reorder(const fg_beam_state& s, const int32_t* parent, const int32_t* len, int nReq, int W) {
  const int64_t units = s.row_bytes * s.rows / (int64_t)sizeof(U);
  const int64_t parts = (int64_t)s.outer * s.inner;
  int64_t gx = (units + kThreads - 1) / kThreads;
  if (gx > 4096) gx = 4096;
#define REORDER(WM)                                                                                                   \
  FG_LAUNCH((beam_reorder_kernel<U, WM>), dim3((unsigned)gx, (unsigned)parts, (unsigned)nReq), dim3(kThreads), 0,     \
            (uint8_t*)s.base, s.beam_stride, s.outer_stride, s.inner, s.inner_stride, s.row_bytes, s.rows, parent, len, \
            W)
  if (W <= 4) REORDER(4);
  else if (W <= 8) REORDER(8);
  else if (W <= 16) REORDER(16);
  else if (W <= 32) REORDER(32);
  else REORDER(64);
#undef REORDER
  return FG_OK;
}

}  // namespace

extern "C" int fg_beam_select(float* score_out, int32_t* token, int32_t* parent, int32_t* done_out,
                              const float* logits, int64_t ld, const float* scores, const int32_t* done, int eos,
                              int nReq, int W, int V) {
  FG_ARG_CHECK(score_out && token && parent && logits && scores, "fg_beam_select: null argument");
  FG_ARG_CHECK(nReq > 0 && V > 0 && W >= 1 && W <= kMaxBeams && nReq <= INT32_MAX / kThreads / W,
               "fg_beam_select: bad dimensions: %d requests, %d beams (1 to %d), vocabulary %d", nReq, W, kMaxBeams, V);
  FG_ARG_CHECK(ld >= V, "fg_beam_select: row stride %lld is below the vocabulary %d", (long long)ld, V);
  FG_ARG_CHECK(!done == !done_out, "fg_beam_select: done and done_out go together");
  FG_ARG_CHECK(eos < V, "fg_beam_select: eos %d outside the vocabulary %d", eos, V);
  FG_ARG_CHECK(!done || eos >= 0, "fg_beam_select: done needs eos");
  const int rows = nReq * W;
  FG_REQUIRE_INIT();
  fg::KProfScope prof("beam_select", 0.0, 4.0 * rows * V);
  fg::Workspace ws;
  const int rc = ws.get((size_t)rows * W * (sizeof(double) + sizeof(int32_t)));
  if (rc != FG_OK) return rc;
  double* val = (double*)ws.ptr;
  int32_t* tok = (int32_t*)(val + (int64_t)rows * W);
  FG_LAUNCH(beam_row_kernel, dim3(rows), dim3(kThreads), 0, val, tok, logits, ld, scores, done, eos, W, V);
  FG_LAUNCH(beam_merge_kernel, dim3(nReq), dim3(64), 0, score_out, token, parent, done_out, (const double*)val,
            (const int32_t*)tok, done, eos, W);
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
    FG_ARG_CHECK(s.outer > 0 && s.inner > 0 && (int64_t)s.outer * s.inner <= 65535 && s.rows >= 0 && s.row_bytes >= 2,
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
  for (int i = 0; i < count; ++i) {
    const fg_beam_state& s = states[i];
    if (s.rows == 0 || W == 1) continue;
    const uintptr_t all = (uintptr_t)s.base | s.beam_stride | s.outer_stride | s.inner_stride | s.row_bytes;
    const int rc = all % 16 == 0 && W <= 32 ? launch_reorder<uint4>(s, parent, len, nReq, W)
                   : all % 8 == 0           ? launch_reorder<uint2>(s, parent, len, nReq, W)
                   : all % 4 == 0           ? launch_reorder<uint32_t>(s, parent, len, nReq, W)
                                            : launch_reorder<uint16_t>(s, parent, len, nReq, W);
    if (rc != FG_OK) return rc;
  }
  return FG_OK;
}
