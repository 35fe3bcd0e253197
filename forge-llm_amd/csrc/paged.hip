// Paged key-value cache (fg_paged_*): storing rows with their positions' rotation,
// reading them back, and causal attention of one or more new tokens a sequence.
#include "common.h"

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
// their angles once.
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
// A wave takes a query of a head, its lanes the head's values.
template <class KV>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(Cache c, int layer, int dH, float* __restrict__ out,
                                                              const float* __restrict__ q, int nH, float scale, int T,
                                                              const int32_t* __restrict__ count, int window, int sinks) {
  const int64_t item = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int64_t row = item / nH;
  const int h = (int)(item - row * nH), lane = threadIdx.x & 63;
  const int s = (int)(row / T), t = (int)(row - (int64_t)s * T);
  if (s >= c.nSeq || t >= new_tokens(count, s, T)) return;
  const int kvh = h / (nH / c.nKV);
  const int64_t pos = (int64_t)slots_used(c, s) + t;
  const int end = (int)min(pos + 1, (int64_t)slots(c));
  const int64_t begin = window > 0 ? pos + 1 - window : 0;  // first slot of the window
  constexpr int N = 4;                                       // values of a lane, up to 256 a head
  float qv[N], o[N] = {}, top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) qv[i] = lane + 64 * i < dH ? q[item * dH + lane + 64 * i] * scale : 0.f;
  for (int j = 0; j < end; ++j) {
    if (j >= sinks && j < begin) j = (int)begin;
    if (j >= end) break;
    const int64_t slot = slot_row(c, layer, s, j);
    if (slot < 0) continue;
    const KV* key = (const KV*)c.k + (slot + ((int64_t)kvh << c.lg)) * dH;
    const KV* val = (const KV*)c.v + (slot + ((int64_t)kvh << c.lg)) * dH;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < dH) d += qv[i] * (float)key[lane + 64 * i];
    d = fg_wave_sum(d);
    const float was = top;
    top = fmaxf(top, d);
    const float keep = was == -INFINITY ? 0.f : expf(was - top), p = expf(d - top);
    sum = sum * keep + p;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < dH) o[i] = o[i] * keep + p * (float)val[lane + 64 * i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 64 * i < dH) out[item * dH + lane + 64 * i] = sum == 0.f ? 0.f : o[i] / sum;
}

// ── entry points' checks ──────────────────────────────────────────────────
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int check_cache(const fg_paged_cache* c, const char* fn) {
  FG_ARG_CHECK(c, "%s: null cache", fn);
  FG_ARG_CHECK(c->nLayers > 0 && c->nSeq > 0 && c->nKvHeads > 0 && c->nPages > 0 && c->maxPages > 0,
               "%s: bad dimensions: %d layers, %d sequences, %d kv heads, %d pages, %d a sequence", fn, c->nLayers,
               c->nSeq, c->nKvHeads, c->nPages, c->maxPages);
  const int d = c->dHead, p = c->pageSize;
  FG_ARG_CHECK(d == 32 || d == 64 || d == 96 || d == 128 || d == 256,
               "%s: head size %d is not one of 32, 64, 96, 128, 256", fn, d);
  FG_ARG_CHECK(p > 0 && p <= 1024 && (p & (p - 1)) == 0, "%s: page size %d is not a power of two up to 1024", fn, p);
  FG_ARG_CHECK((int64_t)c->maxPages * p <= 1 << 30, "%s: %d pages of %d slots a sequence are above 2^30", fn,
               c->maxPages, p);
  FG_ARG_CHECK(c->nKvHeads <= 1 << 16 && (int64_t)c->nLayers * c->nPages < (int64_t)1 << 36,
               "%s: %d layers of %d pages of %d kv heads are too many", fn, c->nLayers, c->nPages, c->nKvHeads);
  FG_ARG_CHECK(c->type == 0 || c->type == 1, "%s: type %d is neither F32 (0) nor F16 (1)", fn, c->type);
  FG_ARG_CHECK(c->k && c->v && c->table && c->len, "%s: null array", fn);
  FG_ARG_CHECK(aligned16(c->k) && aligned16(c->v), "%s: the cache's pages must be 16-byte aligned", fn);
  return FG_OK;
}
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

#define PAGED_TRY(expr)               \
  do {                                \
    const int rc_ = (expr);           \
    if (rc_ != FG_OK) return rc_;     \
  } while (0)

extern "C" int fg_paged_append(const fg_paged_cache* c, int layer, float* q_out, const float* q, const float* k,
                               const float* v, int64_t ld, int nHeads, int T, const int32_t* count,
                               const double* cos_tab, const double* sin_tab, int npos, int rot, int half) {
  const char* fn = "fg_paged_append";
  PAGED_TRY(check_cache(c, fn));
  PAGED_TRY(check_step(c, layer, T, fn));
  FG_ARG_CHECK(T == 0 || (k && v), "%s: null argument", fn);
  FG_ARG_CHECK(!q == !q_out, "%s: q and q_out are given together", fn);
  const int nH = q ? nHeads : 0;
  FG_ARG_CHECK(!q || (nHeads > 0 && nHeads <= 1 << 20), "%s: %d query heads", fn, nHeads);
  const int64_t wide = (int64_t)(nH > c->nKvHeads ? nH : c->nKvHeads) * c->dHead;
  FG_ARG_CHECK(ld >= wide, "%s: row stride %lld is below %lld", fn, (long long)ld, (long long)wide);
  FG_ARG_CHECK(q != q_out || !q || ld == wide, "%s: q in place needs rows of %d x %d", fn, nH, c->dHead);
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
  PAGED_TRY(check_cache(c, fn));
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
  PAGED_TRY(check_cache(c, fn));
  PAGED_TRY(check_step(c, layer, T, fn));
  FG_ARG_CHECK(T == 0 || (out && q), "%s: null argument", fn);
  FG_ARG_CHECK(nHeads > 0 && nHeads % c->nKvHeads == 0, "%s: %d query heads for %d kv heads", fn, nHeads, c->nKvHeads);
  FG_ARG_CHECK(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", fn, window, sinks);
  const int64_t items = (int64_t)c->nSeq * T * nHeads;
  FG_ARG_CHECK(items <= INT32_MAX / kThreads, "%s: %d sequences x %d tokens x %d heads are too many", fn, c->nSeq, T, nHeads);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("paged_attn", 0.0, (double)c->nSeq * c->maxPages * c->pageSize * 2 * row_bytes(c));
  const dim3 grid((unsigned)((items + kWaves - 1) / kWaves));
  if (c->type == 0)
    FG_LAUNCH(paged_attn_kernel<float>, grid, dim3(kThreads), 0, view(c), layer, c->dHead, out, q, nHeads, (float)scale,
              T, count, window, sinks);
  else
    FG_LAUNCH(paged_attn_kernel<_Float16>, grid, dim3(kThreads), 0, view(c), layer, c->dHead, out, q, nHeads,
              (float)scale, T, count, window, sinks);
  return FG_OK;
}

extern "C" int fg_paged_commit(const fg_paged_cache* c, int T, const int32_t* count) {
  PAGED_TRY(check_cache(c, "fg_paged_commit"));
  FG_ARG_CHECK(T >= 0, "fg_paged_commit: T %d is negative", T);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("paged_commit", 0.0, 12.0 * c->nSeq);
  FG_LAUNCH(paged_commit_kernel, dim3((c->nSeq + kThreads - 1) / kThreads), dim3(kThreads), 0, view(c), T, count);
  return FG_OK;
}
