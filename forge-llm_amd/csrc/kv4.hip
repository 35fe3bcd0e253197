// 4-bit key-value cache (fg_kv4_*): storing and reading rows, attention of one
// query token a sequence, and eviction by accumulated attention weight.
//
// A slot of a head is nb = dHead / 32 blocks of 32 values, each d (c - 8) with a
// fp16 step d and codes c of 0..15; the codes' bytes interleave the blocks
// (include/forge_hip.h), so 16 neighbouring lanes of nb bytes cover a slot.
#include "common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ── the cache as kernels see it ───────────────────────────────────────────
struct Cache {
  int nSeq, nKV, maxSeq;
  uint8_t *k, *v;
  _Float16 *kd, *vd;
  int32_t *len, *next;
  float* weight;
  int32_t* pos;
};
// Slot 0 of (layer, sequence, kv head), as a slot number of the whole arrays.
__host__ __device__ __forceinline__ int64_t head_slot(const Cache& c, int layer, int s, int h) {
  return (((int64_t)layer * c.nSeq + s) * c.nKV + h) * c.maxSeq;
}
// New tokens of sequence s, and the slots in use before and after them.
__device__ __forceinline__ int new_tokens(const int32_t* count, int s, int T) {
  return count ? min(max(count[s], 0), T) : T;
}
__device__ __forceinline__ int slots_used(const Cache& c, int s) { return min(max(c.len[s], 0), c.maxSeq); }

// ── store ─────────────────────────────────────────────────────────────────
// Sixteen lanes take a head's slot: lane n holds values 32 b + n and 32 b + 16 + n
// of every block, so a block's maximum is a reduction over 16 lanes and the
// lane's nb bytes are its share of the slot.  floor(x / d + 8.5) is found from
// an approximate quotient and the exact borders (c - 8.5) d: 5 bits times 11
// bits, no rounding in fp32.
__device__ __forceinline__ int code_of(float x, float inv, float d) {
  const float y = d < 0.f ? -x : x, s = fabsf(d);
  float q = floorf(y * inv + 8.5f);
  if (y < (q - 8.5f) * s) q -= 1.f;
  else if (y >= (q - 7.5f) * s) q += 1.f;
  return (int)fminf(fmaxf(q, 0.f), 15.f);
}

template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Cache c, int layer, const float* __restrict__ k,
                                                              const float* __restrict__ v, int64_t ld, int T,
                                                              const int32_t* __restrict__ count, int64_t rows) {
  constexpr int dH = 32 * NB;
  const int n = threadIdx.x & 15, lane0 = threadIdx.x & 48;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
  const bool on = item < rows * c.nKV;
  const int64_t row = on ? item / c.nKV : 0;
  const int h = on ? (int)(item - row * c.nKV) : 0;
  const int s = (int)(row / T), t = (int)(row - (int64_t)s * T);
  const int64_t at = (int64_t)slots_used(c, s) + t;
  if (!on || t >= new_tokens(count, s, T) || at >= c.maxSeq) return;  // whole groups of 16 lanes
  const float* x = (blockIdx.y ? v : k) + row * ld + (int64_t)h * dH;
  const int64_t slot = head_slot(c, layer, s, h) + at;
  float lo[NB], hi[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    lo[b] = x[32 * b + n];
    hi[b] = x[32 * b + 16 + n];
  }
  uint8_t* bytes = (blockIdx.y ? c.v : c.k) + slot * (dH / 2) + n * NB;
  _Float16* steps = (blockIdx.y ? c.vd : c.kd) + slot * NB;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float a = fmaxf(fabsf(lo[b]), fabsf(hi[b]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 16));
    const uint32_t in_lo = (uint32_t)(__ballot(fabsf(lo[b]) == a) >> lane0) & 0xFFFF;
    const uint32_t in_hi = (uint32_t)(__ballot(fabsf(hi[b]) == a) >> lane0) & 0xFFFF;
    const uint32_t neg_lo = (uint32_t)(__ballot(lo[b] < 0.f) >> lane0) & 0xFFFF;
    const uint32_t neg_hi = (uint32_t)(__ballot(hi[b] < 0.f) >> lane0) & 0xFFFF;
    const bool nan = ((uint32_t)(__ballot(lo[b] != lo[b] || hi[b] != hi[b]) >> lane0) & 0xFFFF) != 0;
    const bool neg = in_lo ? (neg_lo >> __builtin_ctz(in_lo)) & 1 : (neg_hi >> __builtin_ctz(in_hi | 0x10000)) & 1;
    _Float16 d = (_Float16)((neg ? a : -a) * 0.125f);  // m / -8
    const float df = (float)d;
    const bool bad = nan || !(fabsf(df) < INFINITY);
    int q0 = 8, q1 = 8;
    if (!bad && df != 0.f) {
      const float inv = 1.f / fabsf(df);
      q0 = code_of(lo[b], inv, df);
      q1 = code_of(hi[b], inv, df);
    }
    bytes[b] = (uint8_t)(q0 | (q1 << 4));
    if (n == 0) steps[b] = bad ? (_Float16)NAN : d;
  }
  if (n == 0 && blockIdx.y == 0) {
    if (c.weight) c.weight[slot] = 0.f;
    if (c.pos) c.pos[slot] = c.next[s] + t;
  }
}

template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Cache c, int layer, float* __restrict__ k,
                                                            float* __restrict__ v, int64_t ld, int first, int T,
                                                            int64_t rows) {
  constexpr int dH = 32 * NB;
  const int n = threadIdx.x & 15;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
  if (item >= rows * c.nKV) return;
  const int64_t row = item / c.nKV;
  const int h = (int)(item - row * c.nKV);
  const int s = (int)(row / T), t = (int)(row - (int64_t)s * T);
  const int64_t slot = head_slot(c, layer, s, h) + first + t;
  const uint8_t* bytes = (blockIdx.y ? c.v : c.k) + slot * (dH / 2) + n * NB;
  const _Float16* steps = (blockIdx.y ? c.vd : c.kd) + slot * NB;
  float* x = (blockIdx.y ? v : k) + row * ld + (int64_t)h * dH;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int q = bytes[b];
    const float d = (float)steps[b];
    x[32 * b + n] = d * (float)((q & 15) - 8);
    x[32 * b + 16 + n] = d * (float)((q >> 4) - 8);
  }
}

// ── attention ─────────────────────────────────────────────────────────────
// Value i of a head's slot.
template <int NB>
__device__ __forceinline__ float value_at(const uint8_t* codes, const _Float16* steps, int64_t slot, int i) {
  const int b = i >> 5, n = i & 15, hi = (i >> 4) & 1;
  const int q = (codes[slot * 16 * NB + n * NB + b] >> (4 * hi)) & 15;
  return (float)steps[slot * NB + b] * (float)(q - 8);
}

__device__ __forceinline__ float block_max(float x, float* sh) {
  x = fg_wave_max(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) x = fmaxf(x, sh[i]);
  return x;
}
__device__ __forceinline__ float block_sum(float x, float* sh) {
  x = fg_wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.f;
  for (int i = 0; i < kWaves; ++i) x += sh[i];
  return x;
}

// One workgroup per (sequence, kv head), a query head after the other: scores
// to `sc`, their maximum and sum, then a value column per thread.
template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(Cache c, int layer, float* __restrict__ out,
                                                            const float* __restrict__ q, int nH, float scale, int T,
                                                            const int32_t* __restrict__ count,
                                                            float* __restrict__ sc) {
  constexpr int dH = 32 * NB;
  __shared__ float sh[kWaves], qs[dH];
  const int s = blockIdx.y, kvh = blockIdx.x, group = nH / c.nKV;
  const int n = min(slots_used(c, s) + new_tokens(count, s, T), c.maxSeq);
  const int64_t slot0 = head_slot(c, layer, s, kvh);
  for (int g = 0; g < group; ++g) {
    const int h = kvh * group + g;
    float* row = sc + ((int64_t)s * nH + h) * c.maxSeq;
    __syncthreads();
    if (threadIdx.x < dH) qs[threadIdx.x] = q[((int64_t)s * nH + h) * dH + threadIdx.x];
    __syncthreads();
    float m = -INFINITY;
    for (int j = threadIdx.x; j < n; j += kThreads) {
      float dot = 0.f;
      for (int i = 0; i < dH; ++i) dot += qs[i] * value_at<NB>(c.k, c.kd, slot0 + j, i);
      row[j] = dot * scale;
      m = fmaxf(m, row[j]);
    }
    m = block_max(m, sh);
    float l = 0.f;
    for (int j = threadIdx.x; j < n; j += kThreads) {
      row[j] = expf(row[j] - m);
      l += row[j];
    }
    l = block_sum(l, sh);
    const float inv = n > 0 ? 1.f / l : 0.f;
    if (c.weight)
      for (int j = threadIdx.x; j < n; j += kThreads) c.weight[slot0 + j] += row[j] * inv;
    __syncthreads();
    if (threadIdx.x < dH) {
      float o = 0.f;
      for (int j = 0; j < n; ++j) o += row[j] * value_at<NB>(c.v, c.vd, slot0 + j, threadIdx.x);
      out[((int64_t)s * nH + h) * dH + threadIdx.x] = o * inv;
    }
  }
}

__global__ void kv4_commit_kernel(Cache c, int T, const int32_t* __restrict__ count) {
  const int s = blockIdx.x * kThreads + threadIdx.x;
  if (s >= c.nSeq) return;
  const int add = new_tokens(count, s, T);
  c.len[s] = min(slots_used(c, s) + add, c.maxSeq);
  c.next[s] += add;
}

// ── eviction ──────────────────────────────────────────────────────────────
// A weight's rank as an unsigned key: NaN lowest, -0 as +0; kept regardless:
// the highest key, which no weight has.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelect = 1024;
// The number of `in` flags of the workgroup's earlier threads; `all` gets the
// number of all.
__device__ __forceinline__ int block_rank(bool in, int* sh, int& all) {
  const unsigned long long b = __ballot(in);
  const int w = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[w] = __popcll(b);
  __syncthreads();
  int before = __popcll(b & ((1ull << (threadIdx.x & 63)) - 1));
  all = 0;
  for (int i = 0; i < kSelect / 64; ++i) {
    if (i < w) before += sh[i];
    all += sh[i];
  }
  return before;
}

// One workgroup per head: the budget-th greatest key by four passes of 8 bits
// over the keys, then the lists in slot order.
__global__ void __launch_bounds__(kSelect) evict_select_kernel(int32_t* __restrict__ holes,
                                                               int32_t* __restrict__ movers,
                                                               int32_t* __restrict__ moves,
                                                               const float* __restrict__ weight,
                                                               const int32_t* __restrict__ pos,
                                                               const int32_t* __restrict__ len,
                                                               const int32_t* __restrict__ next, int nSeq, int nHeads,
                                                               int maxSeq, int budget, int recent, int most) {
  __shared__ int hist[256], sh[kSelect / 64], pick[2];
  const int64_t head = blockIdx.x;
  const int s = (int)(head / nHeads % nSeq);
  const int n = min(max(len[s], 0), maxSeq);
  const int64_t safe = (int64_t)next[s] - recent;
  weight += head * maxSeq;
  pos += head * maxSeq;
  holes += head * most;
  movers += head * most;
  int nh = 0, nm = 0;
  if (n > budget) {
    auto key = [&](int j) { return (int64_t)pos[j] >= safe ? 0xFFFFFFFFu : weight_key(weight[j]); };
    uint32_t prefix = 0;
    int want = budget;  // of the keys that share the prefix so far
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelect) hist[i] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < n; j += kSelect) {
        const uint32_t u = key(j);
        if (shift == 24 || (u >> (shift + 8)) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int i = 255, left = want;
        while (i > 0 && hist[i] < left) left -= hist[i--];
        pick[0] = i;
        pick[1] = left;
      }
      __syncthreads();
      prefix = (prefix << 8) | (uint32_t)pick[0];
      want = pick[1];
      __syncthreads();
    }
    int equals = 0;
    for (int j0 = 0; j0 < n; j0 += kSelect) {
      const int j = j0 + (int)threadIdx.x;
      const uint32_t u = j < n ? key(j) : 0;
      int all;
      const int rank = equals + block_rank(j < n && u == prefix, sh, all);
      equals += all;
      const bool kept = j < n && (u > prefix || (u == prefix && rank < want));
      const bool hole = j < n && j < budget && !kept, mover = kept && j >= budget;
      const int ih = nh + block_rank(hole, sh, all);
      nh += all;
      const int im = nm + block_rank(mover, sh, all);
      nm += all;
      if (hole && ih < most) holes[ih] = j;
      if (mover && im < most) movers[im] = j;
    }
  }
  for (int i = nm + (int)threadIdx.x; i < most; i += kSelect) holes[i] = movers[i] = -1;
  if (threadIdx.x == 0) moves[head] = nm;
}

__global__ void __launch_bounds__(kThreads) kv4_move_kernel(Cache c, const int32_t* __restrict__ holes,
                                                            const int32_t* __restrict__ movers,
                                                            const int32_t* __restrict__ moves, int most, int row,
                                                            int nb) {
  const int64_t head = blockIdx.x;
  const int64_t slot0 = head * c.maxSeq;
  const int n = moves[head];
  for (int i = threadIdx.x >> 6; i < n; i += kWaves) {
    const int64_t to = slot0 + holes[head * most + i], from = slot0 + movers[head * most + i];
    for (int b = threadIdx.x & 63; b < row; b += 64) {
      c.k[to * row + b] = c.k[from * row + b];
      c.v[to * row + b] = c.v[from * row + b];
    }
    for (int b = threadIdx.x & 63; b < nb; b += 64) {
      c.kd[to * nb + b] = c.kd[from * nb + b];
      c.vd[to * nb + b] = c.vd[from * nb + b];
    }
    if ((threadIdx.x & 63) == 0) {
      c.weight[to] = c.weight[from];
      c.pos[to] = c.pos[from];
    }
  }
}

__global__ void kv4_cut_kernel(Cache c, int budget) {
  const int s = blockIdx.x * kThreads + threadIdx.x;
  if (s < c.nSeq) c.len[s] = min(slots_used(c, s), budget);
}

__global__ void kv4_follow_kernel(int32_t* __restrict__ len, int32_t* __restrict__ next,
                                  const int32_t* __restrict__ parent, int W) {
  const int64_t r0 = (int64_t)blockIdx.x * W;
  const int b = threadIdx.x;
  int l = 0, n = 0;
  if (b < W) {
    const int q = parent[r0 + b], p = q >= 0 && q < W ? q : b;
    l = len[r0 + p];
    n = next[r0 + p];
  }
  __syncthreads();
  if (b < W) {
    len[r0 + b] = l;
    next[r0 + b] = n;
  }
}

// ── entry points ──────────────────────────────────────────────────────────
constexpr int kMaxHeads = 1 << 21;  // heads x sequences x layers: a workgroup of 1024 threads each
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

int check_cache(const fg_kv4_cache* c, const char* fn) {
  FG_ARG_CHECK(c, "%s: null cache", fn);
  FG_ARG_CHECK(c->nLayers > 0 && c->nSeq > 0 && c->nKvHeads > 0 && c->maxSeq > 0,
               "%s: bad dimensions: %d layers, %d sequences, %d kv heads, %d slots", fn, c->nLayers, c->nSeq,
               c->nKvHeads, c->maxSeq);
  const int d = c->dHead;
  FG_ARG_CHECK(d == 32 || d == 64 || d == 96 || d == 128 || d == 256,
               "%s: head size %d is not one of 32, 64, 96, 128, 256", fn, d);
  FG_ARG_CHECK((int64_t)c->nLayers * c->nSeq < kMaxHeads / c->nKvHeads, "%s: %d x %d x %d heads are too many", fn,
               c->nLayers, c->nSeq, c->nKvHeads);
  FG_ARG_CHECK(c->k && c->v && c->kd && c->vd && c->len && c->next, "%s: null array", fn);
  FG_ARG_CHECK(aligned16(c->k) && aligned16(c->v) && aligned16(c->kd) && aligned16(c->vd) && aligned16(c->weight) &&
                   aligned16(c->pos),
               "%s: the cache's arrays must be 16-byte aligned", fn);
  return FG_OK;
}
int check_layer(const fg_kv4_cache* c, int layer, const char* fn) {
  FG_ARG_CHECK(layer >= 0 && layer < c->nLayers, "%s: layer %d outside [0, %d)", fn, layer, c->nLayers);
  return FG_OK;
}
Cache view(const fg_kv4_cache* c) {
  return {c->nSeq, c->nKvHeads, c->maxSeq, c->k, c->v, (_Float16*)c->kd, (_Float16*)c->vd, c->len, c->next, c->weight, c->pos};
}
double slot_bytes(const fg_kv4_cache* c) { return (double)c->nKvHeads * (c->dHead + c->dHead / 8); }

#define KV4_DISPATCH(dH, ...)                                  \
  switch (dH) {                                                \
    case 32: { constexpr int NB = 1; __VA_ARGS__; } break;     \
    case 64: { constexpr int NB = 2; __VA_ARGS__; } break;     \
    case 96: { constexpr int NB = 3; __VA_ARGS__; } break;     \
    case 128: { constexpr int NB = 4; __VA_ARGS__; } break;    \
    default: { constexpr int NB = 8; __VA_ARGS__; } break;     \
  }

}  // namespace

#define KV4_TRY(expr)                 \
  do {                                \
    const int rc_ = (expr);           \
    if (rc_ != FG_OK) return rc_;     \
  } while (0)

extern "C" int fg_kv4_append(const fg_kv4_cache* c, int layer, const float* k, const float* v, int64_t ld, int T,
                             const int32_t* count) {
  KV4_TRY(check_cache(c, "fg_kv4_append"));
  KV4_TRY(check_layer(c, layer, "fg_kv4_append"));
  FG_ARG_CHECK(T >= 0, "fg_kv4_append: T %d is negative", T);
  FG_ARG_CHECK(T == 0 || (k && v), "fg_kv4_append: null argument");
  FG_ARG_CHECK(ld >= (int64_t)c->nKvHeads * c->dHead, "fg_kv4_append: row stride %lld is below %d x %d", (long long)ld,
               c->nKvHeads, c->dHead);
  const int64_t rows = (int64_t)c->nSeq * T, blocks = (rows * c->nKvHeads + 15) / 16;
  FG_ARG_CHECK(blocks <= INT32_MAX / kThreads, "fg_kv4_append: %d sequences x %d tokens are too many", c->nSeq, T);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("kv4_append", 0.0, rows * (8.0 * c->nKvHeads * c->dHead + slot_bytes(c)));
  KV4_DISPATCH(c->dHead, FG_LAUNCH(kv4_append_kernel<NB>, dim3((unsigned)blocks, 2), dim3(kThreads), 0, view(c), layer,
                                   k, v, ld, T, count, rows));
  return FG_OK;
}

extern "C" int fg_kv4_read(const fg_kv4_cache* c, int layer, float* k, float* v, int64_t ld, int first, int T) {
  KV4_TRY(check_cache(c, "fg_kv4_read"));
  KV4_TRY(check_layer(c, layer, "fg_kv4_read"));
  FG_ARG_CHECK(first >= 0 && T >= 0 && (int64_t)first + T <= c->maxSeq, "fg_kv4_read: slots [%d, %lld) outside [0, %d)",
               first, (long long)first + T, c->maxSeq);
  FG_ARG_CHECK(T == 0 || (k && v), "fg_kv4_read: null argument");
  FG_ARG_CHECK(ld >= (int64_t)c->nKvHeads * c->dHead, "fg_kv4_read: row stride %lld is below %d x %d", (long long)ld,
               c->nKvHeads, c->dHead);
  const int64_t rows = (int64_t)c->nSeq * T, blocks = (rows * c->nKvHeads + 15) / 16;
  FG_ARG_CHECK(blocks <= INT32_MAX / kThreads, "fg_kv4_read: %d sequences x %d slots are too many", c->nSeq, T);
  FG_REQUIRE_INIT();
  if (T == 0) return FG_OK;
  fg::KProfScope prof("kv4_read", 0.0, rows * (8.0 * c->nKvHeads * c->dHead + slot_bytes(c)));
  KV4_DISPATCH(c->dHead, FG_LAUNCH(kv4_read_kernel<NB>, dim3((unsigned)blocks, 2), dim3(kThreads), 0, view(c), layer, k,
                                   v, ld, first, T, rows));
  return FG_OK;
}

extern "C" int fg_kv4_attn(const fg_kv4_cache* c, int layer, float* out, const float* q, int nHeads, double scale,
                           int T, const int32_t* count) {
  KV4_TRY(check_cache(c, "fg_kv4_attn"));
  KV4_TRY(check_layer(c, layer, "fg_kv4_attn"));
  FG_ARG_CHECK(out && q, "fg_kv4_attn: null argument");
  FG_ARG_CHECK(T >= 0, "fg_kv4_attn: T %d is negative", T);
  FG_ARG_CHECK(nHeads > 0 && nHeads % c->nKvHeads == 0, "fg_kv4_attn: %d query heads for %d kv heads", nHeads,
               c->nKvHeads);
  FG_ARG_CHECK(c->nSeq <= 65535, "fg_kv4_attn: %d sequences are too many", c->nSeq);
  FG_REQUIRE_INIT();
  fg::KProfScope prof("kv4_attn", 0.0, (double)c->nSeq * c->maxSeq * slot_bytes(c));
  fg::Workspace ws;
  KV4_TRY(ws.get((size_t)c->nSeq * nHeads * c->maxSeq * sizeof(float)));
  KV4_DISPATCH(c->dHead, FG_LAUNCH(kv4_attn_kernel<NB>, dim3(c->nKvHeads, c->nSeq), dim3(kThreads), 0, view(c), layer,
                                   out, q, nHeads, (float)scale, T, count, (float*)ws.ptr));
  return FG_OK;
}

extern "C" int fg_kv4_commit(const fg_kv4_cache* c, int T, const int32_t* count) {
  KV4_TRY(check_cache(c, "fg_kv4_commit"));
  FG_ARG_CHECK(T >= 0, "fg_kv4_commit: T %d is negative", T);
  FG_REQUIRE_INIT();
  fg::KProfScope prof("kv4_commit", 0.0, 16.0 * c->nSeq);
  FG_LAUNCH(kv4_commit_kernel, dim3((c->nSeq + kThreads - 1) / kThreads), dim3(kThreads), 0, view(c), T, count);
  return FG_OK;
}

extern "C" int fg_kv_evict_select(int32_t* holes, int32_t* movers, int32_t* moves, const float* weight,
                                  const int32_t* pos, const int32_t* len, const int32_t* next, int nLayers, int nSeq,
                                  int nHeads, int maxSeq, int budget, int recent) {
  FG_ARG_CHECK(holes && movers && moves && weight && pos && len && next, "fg_kv_evict_select: null argument");
  FG_ARG_CHECK(nLayers > 0 && nSeq > 0 && nHeads > 0 && maxSeq > 0 &&
                   (int64_t)nLayers * nSeq < kMaxHeads / nHeads,
               "fg_kv_evict_select: bad dimensions: %d layers, %d sequences, %d heads, %d slots", nLayers, nSeq, nHeads,
               maxSeq);
  FG_ARG_CHECK(budget >= 1 && budget < maxSeq, "fg_kv_evict_select: budget %d outside [1, %d)", budget, maxSeq);
  FG_ARG_CHECK(recent >= 0 && recent <= budget, "fg_kv_evict_select: recent %d outside [0, %d]", recent, budget);
  const int heads = nLayers * nSeq * nHeads, most = budget < maxSeq - budget ? budget : maxSeq - budget;
  FG_REQUIRE_INIT();
  fg::KProfScope prof("kv_evict_select", 0.0, (double)heads * (8.0 * maxSeq + 8.0 * most));
  FG_LAUNCH(evict_select_kernel, dim3(heads), dim3(kSelect), 0, holes, movers, moves, weight, pos, len, next, nSeq,
            nHeads, maxSeq, budget, recent, most);
  return FG_OK;
}

extern "C" int fg_kv4_evict(const fg_kv4_cache* c, int budget, int recent) {
  KV4_TRY(check_cache(c, "fg_kv4_evict"));
  FG_ARG_CHECK(c->weight && c->pos, "fg_kv4_evict: the cache keeps no weights or positions");
  FG_ARG_CHECK(budget >= 1, "fg_kv4_evict: budget %d is below 1", budget);
  FG_ARG_CHECK(recent >= 0 && recent <= budget, "fg_kv4_evict: recent %d outside [0, %d]", recent, budget);
  FG_REQUIRE_INIT();
  if (budget >= c->maxSeq) return FG_OK;
  const int heads = c->nLayers * c->nSeq * c->nKvHeads, most = budget < c->maxSeq - budget ? budget : c->maxSeq - budget;
  fg::Workspace ws;
  KV4_TRY(ws.get((size_t)heads * (2 * (size_t)most + 1) * sizeof(int32_t)));
  int32_t *holes = (int32_t*)ws.ptr, *movers = holes + (int64_t)heads * most, *moves = movers + (int64_t)heads * most;
  KV4_TRY(fg_kv_evict_select(holes, movers, moves, c->weight, c->pos, c->len, c->next, c->nLayers, c->nSeq, c->nKvHeads,
                             c->maxSeq, budget, recent));
  fg::KProfScope prof("kv4_evict", 0.0, (double)c->nLayers * c->nSeq * most * 2 * slot_bytes(c));
  FG_LAUNCH(kv4_move_kernel, dim3(heads), dim3(kThreads), 0, view(c), (const int32_t*)holes, (const int32_t*)movers,
            (const int32_t*)moves, most, c->dHead / 2, c->dHead / 32);
  FG_LAUNCH(kv4_cut_kernel, dim3((c->nSeq + kThreads - 1) / kThreads), dim3(kThreads), 0, view(c), budget);
  return FG_OK;
}

extern "C" int fg_kv4_reorder(const fg_kv4_cache* c, const int32_t* parent, int W) {
  KV4_TRY(check_cache(c, "fg_kv4_reorder"));
  FG_ARG_CHECK(parent, "fg_kv4_reorder: null argument");
  FG_ARG_CHECK(W >= 1 && W <= 64 && c->nSeq % W == 0, "fg_kv4_reorder: %d sequences are not groups of %d beams "
               "(1 to 64)", c->nSeq, W);
  FG_REQUIRE_INIT();
  fg_beam_state st[6];
  int n = 0;
  auto add = [&](void* base, int64_t row) {
    if (!base) return;
    const int64_t head = c->maxSeq * row, seq = c->nKvHeads * head;
    st[n++] = {base, seq, c->nLayers, c->nSeq * seq, c->nKvHeads, head, row, c->maxSeq};
  };
  add(c->k, c->dHead / 2);
  add(c->v, c->dHead / 2);
  add(c->kd, c->dHead / 16);
  add(c->vd, c->dHead / 16);
  add(c->weight, 4);
  add(c->pos, 4);
  KV4_TRY(fg_beam_reorder(st, n, parent, c->len, c->nSeq / W, W));
  FG_LAUNCH(kv4_follow_kernel, dim3(c->nSeq / W), dim3(64), 0, c->len, c->next, parent, W);
  return FG_OK;
}
