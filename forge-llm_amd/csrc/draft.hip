// Verification of drafted tokens (fg_draft_verify).
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

// Over the workgroup; `sh` holds a value a wave.
__device__ __forceinline__ double group_sum(double x, double* sh) {
  x = fg_wave_sum_d(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < kWaves; ++w) x += sh[w];
  return x;
}
__device__ __forceinline__ float group_max(float x, double* sh) {
  x = fg_wave_max(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  x = (float)sh[0];
  for (int w = 1; w < kWaves; ++w) x = fmaxf(x, (float)sh[w]);
  return x;
}
__device__ __forceinline__ int group_min(int x, double* sh) {
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  x = (int)sh[0];
  for (int w = 1; w < kWaves; ++w) x = min(x, (int)sh[w]);
  return x;
}

struct Row {  // softmax of a row: exp((x - top) inv) / sum
  const float* x;
  double top, inv, sum;
  __device__ __forceinline__ double at(int v) const { return exp(((double)x[v] - top) * inv) / sum; }
};
__device__ Row row_of(const float* x, int V, double inv, double* sh) {
  float m = -INFINITY;
  for (int v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, x[v]);
  Row r{x, group_max(m, sh), inv, 0};
  double e = 0;
  for (int v = threadIdx.x; v < V; v += kThreads) e += exp(((double)x[v] - r.top) * inv);
  r.sum = group_sum(e, sh);
  return r;
}

// A workgroup takes a sequence.
__global__ void __launch_bounds__(kThreads) draft_verify_kernel(int32_t* __restrict__ token, int32_t* __restrict__ count,
                                                                const float* __restrict__ logits, int64_t ld,
                                                                const float* __restrict__ draft_logits, int64_t ld_draft,
                                                                const int32_t* __restrict__ draft,
                                                                const int32_t* __restrict__ drafted,
                                                                const float* __restrict__ u, double inv, int D, int V) {
  __shared__ double sh[kWaves];
  __shared__ double reach[kThreads];
  const int s = blockIdx.x;
  const int n = drafted ? min(drafted[s], D) : D;
  int32_t* tok = token + (int64_t)s * (D + 1);
  if (n < 0) {
    for (int t = threadIdx.x; t <= D; t += kThreads) tok[t] = -1;
    if (threadIdx.x == 0) count[s] = 0;
    return;
  }
  int taken = 0, last = -1;
  for (;; ++taken) {
    const float* x = logits + ((int64_t)s * (D + 1) + taken) * ld;
    const bool more = taken < n;
    const int d = more ? draft[(int64_t)s * D + taken] : -1;
    if (inv == 0) {  // the lowest of the greatest
      float m = -INFINITY;
      for (int v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, x[v]);
      m = group_max(m, sh);
      int at = INT32_MAX;
      for (int v = threadIdx.x; v < V; v += kThreads)
        if (x[v] == m) at = min(at, v);
      at = group_min(at, sh);
      last = at == INT32_MAX ? -1 : at;
      if (more && d == last && d >= 0) continue;
      break;
    }
    const Row p = row_of(x, V, inv, sh);
    Row q{nullptr, 0, 0, 0};
    if (more && draft_logits) q = row_of(draft_logits + ((int64_t)s * D + taken) * ld_draft, V, inv, sh);
    const bool in = d >= 0 && d < V;
    if (more && in && (double)u[(int64_t)s * (D + 1) + taken] * (draft_logits ? q.at(d) : 1.0) < p.at(d)) continue;
    // the weights of the tokens, a run of the vocabulary a thread
    const int run = (V + kThreads - 1) / kThreads, v0 = min((int)threadIdx.x * run, V), v1 = min(v0 + run, V);
    auto weight = [&](int v, bool less) {
      const double a = p.at(v);
      if (!less) return a;
      const double b = q.x ? q.at(v) : v == d ? 1.0 : 0.0;
      return fmax(a - b, 0.0);
    };
    bool less = more;
    double all, mine;
    for (;; less = false) {
      mine = 0;
      for (int v = v0; v < v1; ++v) mine += weight(v, less);
      all = group_sum(mine, sh);
      if (all > 0 || !less) break;
    }
    if (!(all > 0) || !(p.sum > 0)) {
      last = -1;
      break;
    }
    __syncthreads();
    reach[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double sum = 0;
      for (int i = 0; i < kThreads; ++i) sum += reach[i], reach[i] = sum;
    }
    __syncthreads();
    const double goal = (double)u[(int64_t)s * (D + 1) + D] * reach[kThreads - 1];
    int at = INT32_MAX, end = INT32_MAX;  // end: -1 - the last token of any weight
    double sum = threadIdx.x ? reach[threadIdx.x - 1] : 0;
    for (int v = v0; v < v1; ++v) {
      const double w = weight(v, less);
      sum += w;
      if (w > 0) end = -1 - v;
      if (w > 0 && sum > goal) {
        at = v;
        break;
      }
    }
    at = group_min(at, sh);
    end = group_min(end, sh);
    last = at != INT32_MAX ? at : -1 - end;
    break;
  }
  for (int t = threadIdx.x; t <= D; t += kThreads) tok[t] = t < taken ? draft[(int64_t)s * D + t] : t == taken ? last : -1;
  if (threadIdx.x == 0) count[s] = taken + 1;
}

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
  FG_REQUIRE_INIT();
  fg::KProfScope prof("draft_verify", 0.0, 4.0 * V * nSeq * (D + 1 + (drawn ? D : 0)));
  FG_LAUNCH(draft_verify_kernel, dim3(nSeq), dim3(kThreads), 0, token, count, logits, ld, drawn ? draft_logits : nullptr,
            ld_draft, draft, drafted, u, temperature == 0 ? 0.0 : 1.0 / temperature, D, V);
  return FG_OK;
}
