// 4-bit key-value cache (fg_kv4_*): storing and reading rows, attention of one
// query token a sequence, and eviction by accumulated attention weight.
//
// A slot of a head is nb = dHead / 32 blocks of 32 values, each d (c - 8) with a
// fp16 step d and codes c of 0..15; the codes' bytes interleave the blocks
// (include/forge_hip.h), so 16 neighbouring lanes of nb bytes cover a slot.
#include "common.h"
#include "f16split.h"

#include <math.h>
#include <type_traits>

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
  bool only_new;  // sequences without new tokens take no part: none of their slots count
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
__device__ __forceinline__ int slots_after(const Cache& c, const int32_t* count, int s, int T) {
  const int used = slots_used(c, s), more = new_tokens(count, s, T);
  return c.only_new && more == 0 ? 0 : used + min(more, c.maxSeq - used);
}

// Maximum, minimum and sum over the 16 lanes of a row, by rotation.
template <int N>
__device__ __forceinline__ float row_turned(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, row_turned<8>(x));
  x = fmaxf(x, row_turned<4>(x));
  x = fmaxf(x, row_turned<2>(x));
  return fmaxf(x, row_turned<1>(x));
}
__device__ __forceinline__ float row_sum(float x) {
  x += row_turned<8>(x);
  x += row_turned<4>(x);
  x += row_turned<2>(x);
  return x + row_turned<1>(x);
}

// ── store ─────────────────────────────────────────────────────────────────
// Sixteen lanes take a head's slot: lane n holds values 32 b + n and 32 b + 16 + n
// of every block, so a block's extremes are reductions over 16 lanes and the
// lane's nb bytes are its share of the slot.  HBM-bound (7.1 B read for 1 written)
// as long as a block costs few instructions: 16384 tokens of 8 heads of 128 43 us
// (3.6 TB/s read and written), reading them back 26 (5.9 TB/s).

// A block by its definition: the first of the greatest magnitudes by ballots, and
// floor(x / d + 8.5) from an approximate quotient and the exact borders (c - 8.5) d:
// 5 bits times 11 bits, no rounding in fp32.
__device__ __forceinline__ int code_of(float x, float inv, float d) {
  const float y = d < 0.f ? -x : x, s = fabsf(d);
  float q = floorf(y * inv + 8.5f);
  if (y < (q - 8.5f) * s) q -= 1.f;
  else if (y >= (q - 7.5f) * s) q += 1.f;
  return (int)fminf(fmaxf(q, 0.f), 15.f);
}
__device__ __noinline__ uint32_t exact_block(float lo, float hi) {  // step << 16 | codes
  const int lane0 = threadIdx.x & 48;
  const float a = row_max(fmaxf(fabsf(lo), fabsf(hi)));
  const uint32_t in_lo = (uint32_t)(__ballot(fabsf(lo) == a) >> lane0) & 0xFFFF;
  const uint32_t in_hi = (uint32_t)(__ballot(fabsf(hi) == a) >> lane0) & 0xFFFF;
  const uint32_t neg_lo = (uint32_t)(__ballot(lo < 0.f) >> lane0) & 0xFFFF;
  const uint32_t neg_hi = (uint32_t)(__ballot(hi < 0.f) >> lane0) & 0xFFFF;
  const bool nan = ((uint32_t)(__ballot(lo != lo || hi != hi) >> lane0) & 0xFFFF) != 0;
  const bool neg = in_lo ? (neg_lo >> __builtin_ctz(in_lo)) & 1 : (neg_hi >> __builtin_ctz(in_hi | 0x10000)) & 1;
  _Float16 d = (_Float16)((neg ? a : -a) * 0.125f);  // m / -8
  const float df = (float)d;
  const bool bad = nan || !(fabsf(df) < INFINITY);
  if (bad) d = (_Float16)NAN;
  int q0 = 8, q1 = 8;
  if (!bad && df != 0.f) {
    const float inv = 1.f / fabsf(df);
    q0 = code_of(lo, inv, df);
    q1 = code_of(hi, inv, df);
  }
  return (uint32_t)__builtin_bit_cast(uint16_t, d) << 16 | (uint32_t)(q0 | (q1 << 4));
}
// The same where no value is NaN, the step is finite and not 0, the extremes differ
// in size and no quotient is near a border; `sure` is false for lanes that this
// cannot tell for.
__device__ __forceinline__ uint32_t quick_block(float lo, float hi, bool& sure) {
  const float most = row_max(fmaxf(lo, hi)), least = -row_max(fmaxf(-lo, -hi));
  const _Float16 d = (_Float16)((most > -least ? most : least) * -0.125f);
  const float inv = __builtin_amdgcn_rcpf((float)d);
  // quotients up to 8.5 (12 for the smallest steps) are off by less than 2^-18
  const float t0 = __builtin_fmaf(lo, inv, 8.5f), t1 = __builtin_fmaf(hi, inv, 8.5f);
  const float f0 = __builtin_amdgcn_fractf(t0), f1 = __builtin_amdgcn_fractf(t1);
  sure = most != -least && inv != 0.f && fmaxf(fabsf(f0 - 0.5f), fabsf(f1 - 0.5f)) < 0.5f - 0x1p-16f &&
         fmaxf(fabsf(t0), fabsf(t1)) < 32.f && lo == lo && hi == hi;
  const uint32_t q0 = (uint32_t)__builtin_amdgcn_fmed3f(t0 - f0, 0.f, 15.f);
  const uint32_t q1 = (uint32_t)__builtin_amdgcn_fmed3f(t1 - f1, 0.f, 15.f);
  return (uint32_t)__builtin_bit_cast(uint16_t, d) << 16 | (q0 | q1 << 4);
}

template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Cache c, int layer, const float* __restrict__ k,
                                                              const float* __restrict__ v, int64_t ld, int T,
                                                              const int32_t* __restrict__ count, uint32_t rows) {
  constexpr int dH = 32 * NB;
  const int n = threadIdx.x & 15;
  const uint32_t item = (blockIdx.x * kThreads + threadIdx.x) >> 4;
  const bool on = item < rows * (uint32_t)c.nKV;
  const uint32_t row = on ? item / (uint32_t)c.nKV : 0;
  const int h = on ? (int)(item - row * (uint32_t)c.nKV) : 0;
  const int s = (int)(row / (uint32_t)T), t = (int)(row - (uint32_t)s * (uint32_t)T);
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
  uint8_t bytes[NB];
  uint16_t steps[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    bool sure;
    uint32_t w = quick_block(lo[b], hi[b], sure);
    if (!__all(sure)) w = exact_block(lo[b], hi[b]);
    bytes[b] = (uint8_t)w;
    steps[b] = (uint16_t)(w >> 16);
  }
  __builtin_memcpy((blockIdx.y ? c.v : c.k) + slot * (dH / 2) + n * NB, bytes, NB);
  if (n == 0) {
    __builtin_memcpy((blockIdx.y ? c.vd : c.kd) + slot * NB, steps, 2 * NB);
    if (blockIdx.y == 0) {
      if (c.weight) c.weight[slot] = 0.f;
      if (c.pos) c.pos[slot] = c.next[s] + t;
    }
  }
}

template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Cache c, int layer, float* __restrict__ k,
                                                            float* __restrict__ v, int64_t ld, int first, int T,
                                                            uint32_t rows) {
  constexpr int dH = 32 * NB;
  const int n = threadIdx.x & 15;
  const uint32_t item = (blockIdx.x * kThreads + threadIdx.x) >> 4;
  if (item >= rows * (uint32_t)c.nKV) return;
  const uint32_t row = item / (uint32_t)c.nKV;
  const int h = (int)(item - row * (uint32_t)c.nKV);
  const int s = (int)(row / (uint32_t)T), t = (int)(row - (uint32_t)s * (uint32_t)T);
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
// One query token a sequence reads the cache once, 1.125 bytes a position and
// head dim for 4 group flop: HBM-bound if decoding the codes costs few enough
// instructions.  Both products run on the fp16 matrix pipes with the codes
// c - 8 as operands, which fp16 holds exactly; what is not exact there is held
// in two fp16 pieces (hi + lo, 22 bits), in rows of their own:
//
//   scores  16 rows (head, piece) of q x 32 values of a block x 16 positions;
//           the block's step multiplies the sum (fp32)
//   values  16 rows (head, piece) of w x 32 positions x 16 values of a block,
//           w = p d with the block's step d, fp32 accumulators
//
// A wave takes 32 positions at a time and keeps the running maximum, sum and
// values of its heads; p = 2^(x - ref) with ref = top + kRoom - 15 + E, 2^E above
// every step so far, so that w stays below 2^15 for scores x up to top + kRoom.
// top (the greatest score) and E are only raised, and the accumulators
// rescaled, when a score or step goes beyond that: with room for a factor of 64
// hardly ever after the first tile (without, four heads of even scores raise
// one's maximum in six of the first ten).  There are eight slots of two rows:
// up to four heads (G) repeat, so that the scores of positions 0 .. 15 come out in
// the lower eight rows and those of 16 .. 31 in the upper, one lane each, and
// 8 / G blocks' steps share an operand of w.
//
// 32 heads on 8 kv heads of 128, 130001 positions 32.3 us (4.6 TB/s) and the join 5.4;
// 32 sequences of up to 8192 40.7 (the last pieces are uneven) and 6.4.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRound = 128;  // positions a workgroup takes at a time, 32 a wave
// Workgroups a CU, by registers.
template <int NB>
constexpr int kResident = NB > 4 ? 2 : NB > 2 ? 3 : 4;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kRoom = 6.f;   // powers of two that a score may pass the maximum by

// How the positions of all sequences are cut: pieces of `per` rounds, at least
// one a sequence and head, `target` of them beside the sequences' last ones.  A
// wave works it out from the lengths (which only the device knows): a lane per
// sequence, or several.
struct Plan {
  int per;
  int s, first, pieces;  // a sequence, its first piece (of one head) and their number
};
__device__ __forceinline__ int rounds_of(int n) { return (n + kRound - 1) / kRound; }
__device__ __forceinline__ int pieces_of(int n, int per) { return max(1, (rounds_of(n) + per - 1) / per); }
// The sequence with the piece id / heads (by_seq false), or sequence id.  False
// if there is no such piece.
__device__ __forceinline__ bool plan_for(Plan& p, const Cache& c, const int32_t* count, int T, int heads, int target,
                                         int id, bool by_seq) {
  if (c.nSeq == 1) {
    const int r = rounds_of(slots_after(c, count, 0, T));
    p.per = (int)max((int64_t)1, ((int64_t)r * heads + target - 1) / target);
    p.s = p.first = 0;
    p.pieces = max(1, (r + p.per - 1) / p.per);
    return by_seq || id < (int64_t)p.pieces * heads;
  }
  const int lane = threadIdx.x & 63, each = (c.nSeq + 63) / 64, s0 = lane * each;
  int64_t rounds = 0;
  for (int i = 0; i < each && s0 + i < c.nSeq; ++i) rounds += rounds_of(slots_after(c, count, s0 + i, T));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) rounds += __shfl_xor(rounds, o, 64);
  p.per = (int)max((int64_t)1, (rounds * heads + target - 1) / target);
  int mine = 0;
  for (int i = 0; i < each && s0 + i < c.nSeq; ++i) mine += pieces_of(slots_after(c, count, s0 + i, T), p.per);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(upto, o, 64);
    if (lane >= o) upto += u;
  }
  const unsigned long long has = __ballot(by_seq ? id < s0 + each : id < (int64_t)upto * heads);
  if (!has) return false;
  const int owner = __builtin_ctzll(has);
  p.s = owner * each;
  p.first = __shfl(upto - mine, owner, 64);
  for (;; ++p.s) {
    p.pieces = pieces_of(slots_after(c, count, p.s, T), p.per);
    if (by_seq ? p.s == id : id < (int64_t)(p.first + p.pieces) * heads) return true;
    p.first += p.pieces;
  }
}

// The low and the high codes of a byte pair, less 8: 0x6400 | c is the fp16
// 1024 + c, and 0x6400 | 16 c is 1024 + 16 c.  `magic` is 0x64006400 in a vector
// register, so that mask and or are one instruction (one scalar operand each).
__device__ __forceinline__ uint32_t low_codes(uint32_t x, uint32_t magic) {
  const f16x2 y = __builtin_bit_cast(f16x2, (x & 0x000F000Fu) | magic) + (f16x2){-1032.f, -1032.f};
  return __builtin_bit_cast(uint32_t, y);
}
__device__ __forceinline__ uint32_t high_codes(uint32_t x, uint32_t magic) {
  const f16x2 y = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (x & 0x00F000F0u) | magic),
                                            (f16x2){0.0625f, 0.0625f}, (f16x2){-72.f, -72.f});
  return __builtin_bit_cast(uint32_t, y);
}
__device__ __forceinline__ f16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(f16x8, (u32x4){a, b, c, d});
}
// N bytes from p, at any alignment, as words.
template <int N>
__device__ __forceinline__ void load_bytes(uint32_t (&w)[(N + 3) / 4], const void* p) {
  w[(N + 3) / 4 - 1] = 0;
  __builtin_memcpy(w, p, N);
}
__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return (float)__builtin_bit_cast(f16x2, w)[i];
}

// 32 positions of a head's cache, as a lane of a wave holds them: lane
// (i = lane & 15, g = lane >> 4) has values 4 g .. 4 g + 3 and 16 more on of every
// block of positions i and 16 + i's keys, and values i and 16 + i of every block
// of positions 4 e + g, e < 8: a load of the wave is a run of the array.  The
// values' steps come in once, half a position's a lane.  Loads start at the tile's first slot (uniform); `left` of its positions exist
// (1 or more), the rest repeat the last.
template <bool Whole>
__device__ __forceinline__ uint32_t tile_slot(int j, int left) {
  return (uint32_t)(Whole ? j : min(j, left - 1));
}
template <int NB, bool Halves>
struct KeyTile {
  uint32_t k[2][NB];                          // bytes j NB + b: value 4 g + j of block b
  uint32_t kd[Halves ? 1 : 2][(NB + 1) / 2];  // steps, of position 16 (g / 2) + i where halved
  template <bool Whole>
  __device__ __forceinline__ void load(const Cache& c, int64_t slot, int left) {
    const uint8_t *bk = c.k + slot * (16 * NB), *dk = (const uint8_t*)(c.kd + slot * NB);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t j = tile_slot<Whole>(Whole ? i : 16 * t + i, left), imm = Whole ? 16 * t : 0;
      load_bytes<4 * NB>(k[t], bk + (j * (16 * NB) + g * 4 * NB) + imm * (16 * NB));
      if constexpr (!Halves) load_bytes<2 * NB>(kd[t], dk + j * (2 * NB) + imm * (2 * NB));
    }
    if constexpr (Halves) load_bytes<2 * NB>(kd[0], dk + tile_slot<Whole>(16 * (g >> 1) + i, left) * (2 * NB));
  }
};
template <int NB>
struct ValueTile {
  uint32_t v[8][(NB + 3) / 4];       // byte b
  uint32_t d[NB == 8 ? 2 : 1];       // steps
  template <bool Whole>
  __device__ __forceinline__ void load(const Cache& c, int64_t slot, int left) {
    const uint8_t *bv = c.v + slot * (16 * NB), *dv = (const uint8_t*)(c.vd + slot * NB);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t j = tile_slot<Whole>(Whole ? g : 4 * e + g, left), imm = Whole ? 4 * e : 0;
      load_bytes<NB>(v[e], bv + (j * (16 * NB) + i * NB) + imm * (16 * NB));
    }
    // a lane takes half of a position's steps, of three the first or last two
    constexpr int H = NB == 1 ? 1 : (NB + 1) / 2;
    load_bytes<2 * H>(d, dv + tile_slot<Whole>(lane >> 1, left) * (2 * NB) + (lane & 1) * (NB - H) * 2);
  }
};

// Over the wave.
__device__ __forceinline__ float lane_value(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}
__device__ __forceinline__ float wave_max(float x) {
  x = row_max(x);
  return fmaxf(fmaxf(lane_value(x, 0), lane_value(x, 16)), fmaxf(lane_value(x, 32), lane_value(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = row_sum(x);
  return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

// Waves of a workgroup that has all of a head, as many as the LDS takes.
template <int NB, int G>
constexpr int kWholeWaves = NB * G > 32 ? 4 : 8;

// G heads (1, 2, 4 or 8) of a kv head, or of a share of its query heads, over one
// piece of a sequence.  Pieces that are a whole sequence give the output, others
// their reference, sum and values.  Whole: one workgroup a sequence and head, no
// plan, no pieces; it adds the weights, too (sc != NULL), from the scores that it
// has left in sc.
template <int NB, int G, bool Whole>
__global__ void __launch_bounds__((Whole ? 64 * kWholeWaves<NB, G> : kThreads), (Whole ? 2 : kResident<NB>)) kv4_attn_kernel(
    Cache c, int layer, float* __restrict__ out, const float* __restrict__ q, int nH, int subs, float scale, int T,
    const int32_t* __restrict__ count, int target, float2* __restrict__ part_ml, float* __restrict__ part_o,
    float* __restrict__ sc) {
  constexpr int dH = 32 * NB, NS = 8 / G, NA = (NB + NS - 1) / NS;  // sets of rows, blocks of a set
  constexpr int kHalves = G <= 4 ? 2 : 1, kScores = 2 / kHalves;     // a lane's positions of a tile
  constexpr int kW = Whole ? kWholeWaves<NB, G> : kWaves, kStep = 32 * kW;
  __shared__ __attribute__((aligned(16))) float ps[kW][G][32];
  __shared__ __attribute__((aligned(16))) _Float16 ds[kW][4][NB][8];
  // q's operand at first, the waves' values at the end
  constexpr int kShared = kW * G * dH > NB * 64 * 4 ? kW * G * dH : NB * 64 * 4;
  __shared__ __attribute__((aligned(16))) float shared[kShared];
  float(*const os)[G][dH] = reinterpret_cast<float(*)[G][dH]>(shared);  // [kW]
  u32x4(*const qs)[64] = reinterpret_cast<u32x4(*)[64]>(shared);        // [NB]
  __shared__ float ms[kW][G], ls[kW][G], qm[kW][16];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int s, head, begin, n, end, pieces;  // head: (kv head, share of its query heads)
  if constexpr (Whole) {
    s = blockIdx.x / (c.nKV * subs);
    head = blockIdx.x - s * (c.nKV * subs);
    n = end = slots_after(c, count, s, T);
    begin = 0;
    pieces = 1;
  } else {
    Plan p;
    if (!plan_for(p, c, count, T, c.nKV * subs, target, blockIdx.x, false)) return;
    const int per = __builtin_amdgcn_readfirstlane(p.per);
    pieces = __builtin_amdgcn_readfirstlane(p.pieces);
    s = __builtin_amdgcn_readfirstlane(p.s);
    const int in_seq = blockIdx.x - __builtin_amdgcn_readfirstlane(p.first) * c.nKV * subs;
    head = in_seq / pieces;
    n = slots_after(c, count, s, T);
    begin = (in_seq - head * pieces) * per * kRound;
    end = min(n, begin + per * kRound);
  }
  const int kvh = head / subs, sub = head - kvh * subs;
  const int group = nH / c.nKV, share = (group + subs - 1) / subs;
  const int h0 = kvh * group + sub * share, heads = min(share, group - sub * share);
  const int64_t slot0 = head_slot(c, layer, s, kvh);

  const int set = (i >> 1) / G;  // this row's blocks: set NA ..
  KeyTile<NB, kHalves == 2> keys;
  ValueTile<NB> vals;
  int at = begin + 32 * wave;
  if (at + 32 <= end) {
    keys.template load<true>(c, slot0 + at, 32);
    vals.template load<true>(c, slot0 + at, 32);
  }

  // q as the scores' first operand: row = lane & 15 holds slot row / 2, that is
  // head (row / 2) % G, piece row & 1; its head's power 2^-e goes into the scores.
  // The waves share the blocks out.
  f16x8 qa[kHalves][NB];
  float factor[2];
  {
    constexpr int mine = (NB + kW - 1) / kW;
    const int h = (i >> 1) % G;
    const float* qr = q + ((int64_t)s * nH + h0 + min(h, heads - 1)) * dH + 4 * g;
    float x[mine][8];
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < mine; ++k) {
      const int b = min(wave + k * kW, NB - 1);
      __builtin_memcpy(&x[k][0], qr + 32 * b, 16);
      __builtin_memcpy(&x[k][4], qr + 32 * b + 16, 16);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[k][e]));
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (lane < 16) qm[wave][i] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kW; ++w) m = fmaxf(m, qm[w][i]);
    const int e = fg::exponent_of_max(m);
#pragma unroll
    for (int k = 0; k < mine; ++k) {
      const int b = wave + k * kW;
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // operand pairs: values (0, 1), (16, 17), (2, 3), (18, 19) of 4 g
        const int at = (j & 1) * 4 + (j >> 1) * 2;
        uint32_t hi, lo;
        fg::split2h(x[k][at], x[k][at + 1], e, hi, lo);
        w[j] = (i & 1) ? lo : hi;
      }
      if (b < NB) qs[b][lane] = w;
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const u32x4 w = qs[b][lane], none = {0u, 0u, 0u, 0u};
      if constexpr (kHalves == 2) {
        qa[0][b] = __builtin_bit_cast(f16x8, i < 8 ? w : none);
        qa[1][b] = __builtin_bit_cast(f16x8, i < 8 ? none : w);
      } else {
        qa[0][b] = __builtin_bit_cast(f16x8, w);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      factor[j] = __builtin_amdgcn_ldexpf(scale * kLog2e, -__shfl(e, 2 * ((2 * g + j) % G), 64));
  }

  f32x4 o[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b][0] = o[b][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float top[2] = {-INFINITY, -INFINITY}, roof[2] = {-INFINITY, -INFINITY}, ref[2] = {-INFINITY, -INFINITY};
  float sum[2] = {0.f, 0.f};
  int E = -24;
  uint32_t limit = 0;  // the greatest fp16 below 2^E, as its bits
  const float piece_of = (i & 1) ? 1.f : 0.f;
  uint32_t magic = 0x64006400u;
  asm("" : "+v"(magic));

  // scores of positions 16 t + i (of four heads or fewer: 16 (g / 2) + i) for heads
  // (2 g + j) % G, in powers of two
  float x[kScores][2];
  const int i0 = kHalves == 2 ? 16 * (g >> 1) + i : i;
  const bool owns[2] = {(kHalves == 2 ? 2 * (g & 1) : 2 * g) < G, (kHalves == 2 ? 2 * (g & 1) + 1 : 2 * g + 1) < G};
  auto score = [&](int at, auto is_whole) __attribute__((always_inline)) {
    constexpr bool whole = decltype(is_whole)::value;
#pragma unroll
    for (int u = 0; u < kScores; ++u) x[u][0] = x[u][1] = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // the words that hold byte b of values 4 g + 0, 1 and 4 g + 2, 3
        auto pair = [&](int j0) {
          const int a0 = j0 * NB + b, a1 = (j0 + 1) * NB + b;
          return __builtin_amdgcn_perm(keys.k[t][a1 / 4], keys.k[t][a0 / 4], 0x0c000c00u | ((4 + a1 % 4) << 16) | (a0 % 4));
        };
        const uint32_t k01 = pair(0), k23 = pair(2);
        const f16x8 kb = operand(low_codes(k01, magic), high_codes(k01, magic), low_codes(k23, magic), high_codes(k23, magic));
        if (kHalves == 1 && t == 1) d = (f32x4){0.f, 0.f, 0.f, 0.f};
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[kHalves == 2 ? t : 0][b], kb, d, 0, 0, 0);
        if (kHalves == 2 && t == 0) continue;
        const int u = kHalves == 2 ? 0 : t;
        const float step = half_of(keys.kd[u][b / 2], b & 1);
        x[u][0] += (d[0] + d[1]) * step;
        x[u][1] += (d[2] + d[3]) * step;
      }
    }
#pragma unroll
    for (int u = 0; u < kScores; ++u) {
      x[u][0] *= factor[0];
      x[u][1] *= factor[1];
      if (!whole && at + 16 * u + i0 >= end) x[u][0] = x[u][1] = -INFINITY;
    }
  };
  auto add = [&](int at, auto is_whole) __attribute__((always_inline)) {
    constexpr bool whole = decltype(is_whole)::value;
    // raise the maximum or the steps' power where this tile goes beyond them
    uint32_t far = 0;
#pragma unroll
    for (int w = 0; w < (NB == 8 ? 2 : 1); ++w) {
      const uint32_t a = vals.d[w] & 0x7FFF7FFFu, a0 = a & 0xFFFF, a1 = a >> 16;
      far = max(far, max(a0 < 0x7C00 ? a0 : 0u, a1 < 0x7C00 ? a1 : 0u));
    }
    const float here[2] = {fmaxf(x[0][0], x[kScores - 1][0]), fmaxf(x[0][1], x[kScores - 1][1])};
    if (__any(here[0] > roof[0] || here[1] > roof[1] || far > limit)) {
      float f = (float)__builtin_bit_cast(_Float16, (uint16_t)far);
      f = wave_max(f);
      if (f > 0.f) E = max(E, __builtin_amdgcn_frexp_expf(f));
      limit = E > -14 ? (uint32_t)((E + 14) << 10) | 0x3FF : (1u << (E + 24)) - 1;
      float turn[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = row_max(here[j]);
        if constexpr (kHalves == 2) m = fmaxf(m, __shfl_xor(m, 32, 64));
        top[j] = fmaxf(top[j], m);
        roof[j] = top[j] + kRoom;
        const float r = roof[j] + (float)(E - 15);
        turn[j] = r == ref[j] ? 1.f : __builtin_amdgcn_exp2f(ref[j] - r);
        ref[j] = r;
        sum[j] *= turn[j];
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          o[b][u][0] *= turn[0];
          o[b][u][1] *= turn[0];
          o[b][u][2] *= turn[1];
          o[b][u][3] *= turn[1];
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int h = (2 * g + j) % G;
#pragma unroll
      for (int u = 0; u < kScores; ++u) {
        if (sc && owns[j] && h < heads && (whole || at + 16 * u + i0 < end))
          sc[((int64_t)s * nH + h0 + h) * c.maxSeq + at + 16 * u + i0] = x[u][j];
        const float e = __builtin_amdgcn_exp2f(x[u][j] - ref[j]);
        sum[j] += e;
        if (owns[j]) ps[wave][h][8 * (i0 & 3) + 4 * u + (i0 >> 2)] = e;
      }
    }
    // the steps by (position & 3, block, position / 4)
    {
      constexpr int H = NB == 1 ? 1 : (NB + 1) / 2;
      const int at = lane >> 1, first = (lane & 1) * (NB - H);
#pragma unroll
      for (int k = 0; k < H; ++k)
        ds[wave][at & 3][first + k][at >> 2] = __builtin_bit_cast(f16x2, vals.d[k / 2])[k & 1];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float e[8];
    {
      const float4* pr = reinterpret_cast<const float4*>(&ps[wave][(i >> 1) % G][8 * g]);
      const float4 a = pr[0], b = pr[1];
      e[0] = a.x, e[1] = a.y, e[2] = a.z, e[3] = a.w, e[4] = b.x, e[5] = b.y, e[6] = b.z, e[7] = b.w;
    }
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      // w = p d of block a of this row's set, the row's piece of it
      const f16x8 step = *reinterpret_cast<const f16x8*>(&ds[wave][g][min(set * NA + a, NB - 1)][0]);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) y[k] = __builtin_fmaf(e[2 * j + k], (float)step[2 * j + k], 0.f);
        const f16x2 h = __builtin_convertvector((f32x2){y[0], y[1]}, f16x2);
        const f16x2 r = __builtin_convertvector((f32x2){y[0] - piece_of * (float)h[0], y[1] - piece_of * (float)h[1]}, f16x2);
        w[j] = __builtin_bit_cast(uint32_t, r);
      }
      const f16x8 wa = operand(w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int z = 0; z < NS; ++z) {
        const int b = z * NA + a;
        if (b >= NB) break;
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t two = __builtin_amdgcn_perm(vals.v[2 * j + 1][b / 4], vals.v[2 * j][b / 4],
                                                     0x0c000c00u | ((4 + b % 4) << 16) | (b % 4));
          lo[j] = low_codes(two, magic);
          hi[j] = high_codes(two, magic);
        }
        o[b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, operand(lo[0], lo[1], lo[2], lo[3]), o[b][0], 0, 0, 0);
        o[b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, operand(hi[0], hi[1], hi[2], hi[3]), o[b][1], 0, 0, 0);
      }
    }
  };
  // the next tile's keys are fetched once this one's scores are there, its values
  // once this one's are added
  const std::true_type whole;
  const std::false_type part;
  for (; at + 32 <= end; at += kStep) {
    const bool more = at + kStep + 32 <= end;
    score(at, whole);
    if (more) keys.template load<true>(c, slot0 + at + kStep, 32);
    add(at, whole);
    if (more) vals.template load<true>(c, slot0 + at + kStep, 32);
  }
  if (at < end) {
    keys.template load<false>(c, slot0 + at, n - at);
    vals.template load<false>(c, slot0 + at, n - at);
    score(at, part);
    add(at, part);
  }

  // the waves' results joined: references to their maximum, then sums
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    sum[j] = row_sum(sum[j]);
    if constexpr (kHalves == 2) sum[j] += __shfl_xor(sum[j], 32, 64);
    if (i == 0 && 2 * g + j < G) ms[wave][2 * g + j] = ref[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int h = (2 * g + j) % G;
    float m = ms[0][h];
#pragma unroll
    for (int w = 1; w < kW; ++w) m = fmaxf(m, ms[w][h]);
    const float turn = ref[j] == m ? 1.f : __builtin_amdgcn_exp2f(ref[j] - m);
    if (i == 0 && 2 * g + j < G) ls[wave][h] = sum[j] * turn;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if ((2 * g + j) / G == b / NA) os[wave][h][32 * b + 16 * u + i] = (o[b][u][2 * j] + o[b][u][2 * j + 1]) * turn;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < heads * dH; k += 64 * kW) {
    const int h = k / dH, d = k - h * dH;
    float v = 0.f, l = 0.f, m = ms[0][h];
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      v += os[w][h][d];
      l += ls[w][h];
      m = fmaxf(m, ms[w][h]);
    }
    if (pieces == 1) out[((int64_t)s * nH + h0 + h) * dH + d] = n > 0 ? v / l : 0.f;
    else part_o[((int64_t)blockIdx.x * G + h) * dH + d] = v;
    if constexpr (!Whole) {
      if (d == 0 && part_ml) part_ml[(int64_t)blockIdx.x * G + h] = make_float2(m, l);
    }
  }
  if constexpr (Whole) {
    if (!sc) return;
    float m[G], inv[G];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      m[h] = ms[0][h];
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        m[h] = fmaxf(m[h], ms[w][h]);
        l += ls[w][h];
      }
      inv[h] = 1.f / l;
    }
    for (int j = threadIdx.x; j < n; j += 64 * kW) {
      float add = 0.f;
#pragma unroll
      for (int h = 0; h < G; ++h)
        if (h < heads) add += __builtin_amdgcn_exp2f(sc[((int64_t)s * nH + h0 + h) * c.maxSeq + j] - m[h]) * inv[h];
      c.weight[slot0 + j] += add;
    }
  }
}

// The pieces of every sequence joined: workgroups [0, nSeq nH) the output of a query
// head, the rest (weights kept) the weights of kJoin positions of a kv head.
// Short launches, so loads that do not depend on each other go first: a head's
// values of its first pieces beside its references, the scores beside them.
constexpr int kJoinPieces = 1024;  // pieces whose factors are kept in LDS
// Reference and sum of a head over its pieces, by one wave; w gets the pieces'
// factors.
__device__ __forceinline__ float2 join_head(const float2* __restrict__ ml, int G, int pieces, float* w) {
  const int lane = threadIdx.x & 63;
  float2 first = make_float2(-INFINITY, 0.f);
  if (lane < pieces) first = ml[(int64_t)lane * G];
  float m = first.x;
  for (int k = lane + 64; k < pieces; k += 64) m = fmaxf(m, ml[(int64_t)k * G].x);
  m = wave_max(m);
  float l = 0.f;
  for (int k = lane; k < pieces; k += 64) {
    const float2 v = k == lane ? first : ml[(int64_t)k * G];
    const float f = v.x == m ? 1.f : __builtin_amdgcn_exp2f(v.x - m);
    if (w && k < kJoinPieces) w[k] = f;
    l += v.y * f;
  }
  return make_float2(m, wave_sum(l));
}

template <int NB, int kJoin>  // threads, and positions of a weights' workgroup
__global__ void __launch_bounds__(kJoin) kv4_join_kernel(Cache c, int layer, float* __restrict__ out, int nH, int subs,
                                                         int G, int T, const int32_t* __restrict__ count, int target,
                                                         const float2* __restrict__ part_ml,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ sc, int chunks) {
  constexpr int dH = 32 * NB, kLanes = kJoin / dH, kAhead = 4096 / kJoin, kJoinWaves = kJoin / 64;
  __shared__ float red[kJoin], factor[kJoinPieces], shm[kJoinWaves], shl[kJoinWaves];
  const int group = nH / c.nKV, share = (group + subs - 1) / subs;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool weights = (int)blockIdx.x >= c.nSeq * nH;
  const int id = weights ? blockIdx.x - c.nSeq * nH : blockIdx.x;
  const int s = weights ? id / (c.nKV * chunks) : id / nH;
  Plan p;
  plan_for(p, c, count, T, c.nKV * subs, target, s, true);
  auto first_of = [&](int kvh, int r) {  // of query head r of its group
    return ((int64_t)p.first * c.nKV * subs + (int64_t)(kvh * subs + r / share) * p.pieces) * G + r % share;
  };
  if (weights) {
    const int n = slots_after(c, count, s, T), kvh = id / chunks % c.nKV, at = id % chunks * kJoin + (int)threadIdx.x;
    if (id % chunks * kJoin >= n) return;
    float sum = 0.f;
    for (int h0 = 0; h0 < group; h0 += 4) {
      float x[4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
        x[h] = h0 + h < group && at < n ? sc[((int64_t)s * nH + kvh * group + h0 + h) * c.maxSeq + at] : 0.f;
      __syncthreads();
      if (wave < 4 && h0 + wave < group) {
        const float2 v = join_head(part_ml + first_of(kvh, h0 + wave), G, p.pieces, nullptr);
        shm[wave] = v.x;
        shl[wave] = 1.f / v.y;
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (h0 + h < group) sum += __builtin_amdgcn_exp2f(x[h] - shm[h]) * shl[h];
    }
    if (at < n) c.weight[head_slot(c, layer, s, kvh) + at] += sum;
    return;
  }
  if (p.pieces == 1) return;
  const int h = id % nH, kvh = h / group;
  const int64_t first = first_of(kvh, h - kvh * group);
  const int d = threadIdx.x % dH, z = threadIdx.x / dH;
  const float* po = part_o + first * dH + d;
  const int64_t step = (int64_t)G * dH;
  float ahead[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int k = z + u * kLanes;
    ahead[u] = z < kLanes && k < p.pieces ? po[k * step] : 0.f;
  }
  if (wave == 0) {
    const float2 ml = join_head(part_ml + first, G, p.pieces, factor);
    shm[0] = ml.x;
    shl[0] = ml.y;
  }
  __syncthreads();
  const float m = shm[0];
  auto turn = [&](int k) {
    if (k < kJoinPieces) return factor[k];
    const float mk = part_ml[first + (int64_t)k * G].x;
    return mk == m ? 1.f : __builtin_amdgcn_exp2f(mk - m);
  };
  float v = 0.f;
  if (z < kLanes) {
    for (int k0 = z; k0 < p.pieces; k0 += kAhead * kLanes) {
      if (k0 != z) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          ahead[u] = k0 + u * kLanes < p.pieces ? po[(k0 + u * kLanes) * step] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (k0 + u * kLanes < p.pieces) v += ahead[u] * turn(k0 + u * kLanes);
    }
  }
  red[threadIdx.x] = v;
  __syncthreads();
  if (z == 0) {
    for (int k = 1; k < kLanes; ++k) v += red[k * dH + d];
    out[((int64_t)s * nH + h) * dH + d] = v / shl[0];
  }
}

__global__ void kv4_commit_kernel(Cache c, int T, const int32_t* __restrict__ count) {
  const int s = blockIdx.x * kThreads + threadIdx.x;
  if (s >= c.nSeq) return;
  c.len[s] = slots_after(c, count, s, T);
  c.next[s] += new_tokens(count, s, T);
}

// ── eviction ──────────────────────────────────────────────────────────────
// A weight's rank as an unsigned key: NaN lowest, -0 as +0; kept regardless:
// the highest key, which no weight has.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64;
constexpr int kBinBits = 11, kBins = 1 << kBinBits;  // two bins a thread
static_assert(kBins == 2 * kSelect, "every bin has a thread");

// The sum of x over the workgroup's later threads; `all` gets the sum of all.
__device__ __forceinline__ int sum_after(int x, int* sh, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_down(s, o, 64);
    if (lane + o < 64) s += u;
  }
  __syncthreads();
  if (lane == 0) sh[w] = s;
  __syncthreads();
  s -= x;
  all = 0;
  for (int i = 0; i < kSelectWaves; ++i) {
    all += sh[i];
    if (i > w) s += sh[i];
  }
  return s;
}

// One workgroup per head.  The keys are cut into 2048 bins by their leading bits,
// quarters of a power of two, and the bin that the budget ends in is found from the
// counts; its keys, one a thread when they are few enough, are cut again until all or
// equals of them are kept.  Weights spread over many powers of two, so a histogram of
// keys is flat where one of the exponent byte piles up (256 heads of 16384 slots:
// four passes of 8 bits took 93 us).
//
// Kept: keys above `border`, and the first `take` of those equal to it.
constexpr uint32_t kSafe = 0xFFFFFFFFu;
struct Search {
  int bins[kBins], sh[kSelectWaves], kept_by_wave[kSelectWaves], pick[3];
  uint32_t list[kSelect];
};
template <class AllKeys>  // all_keys(take): take(u) for every key of this thread
__device__ __forceinline__ void find_border(AllKeys all_keys, int budget, Search& f, uint32_t& border, int& take) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int want = 0;  // of the keys in [lo, hi]
  uint32_t lo = 0, hi = kSafe - 1;
  // the bin of [lo, hi] that the want-th greatest of its keys is in becomes
  // [lo, hi], `want` counts inside it; its number of keys
  auto narrow = [&](auto first, auto each_key) {
    const int shift = max(0, 32 - kBinBits - (int)__builtin_clz(hi - lo));
    for (int i = threadIdx.x; i < kBins; i += kSelect) f.bins[i] = 0;
    __syncthreads();
    int safes = 0;
    each_key([&](uint32_t u) {
      if (decltype(first)::value) safes += u == kSafe;
      if (u >= lo && u <= hi) atomicAdd(&f.bins[(u - lo) >> shift], 1);
    });
    if constexpr (decltype(first)::value) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) safes += __shfl_xor(safes, o, 64);
      if (lane == 0) f.kept_by_wave[wave] = safes;
    }
    __syncthreads();
    if constexpr (decltype(first)::value) {
      want = budget;
      for (int w = 0; w < kSelectWaves; ++w) want -= f.kept_by_wave[w];
      if (want <= 0) return want;
    }
    const int b0 = f.bins[2 * threadIdx.x], b1 = f.bins[2 * threadIdx.x + 1];
    int all;
    const int after = sum_after(b0 + b1, f.sh, all);
    if (after < want && want <= after + b0 + b1) {
      const bool upper = want <= after + b1;
      f.pick[0] = 2 * threadIdx.x + upper;
      f.pick[1] = want - after - (upper ? 0 : b1);
      f.pick[2] = upper ? b1 : b0;
    }
    __syncthreads();
    lo += (uint32_t)f.pick[0] << shift;
    hi = min(hi, lo + ((1u << shift) - 1));
    want = f.pick[1];
    return f.pick[2];
  };
  const std::true_type first;
  const std::false_type later;
  int c = narrow(first, all_keys);
  // three levels of 11 bits make lo == hi
  for (int level = 1; level < 3 && want > 0 && lo != hi && c != want && c > kSelect; ++level) c = narrow(later, all_keys);
  if (want > 0 && lo != hi && c != want) {
    // few enough to hold one a thread
    __syncthreads();
    if (threadIdx.x == 0) f.pick[2] = 0;
    __syncthreads();
    all_keys([&](uint32_t u) {
      if (u >= lo && u <= hi) f.list[atomicAdd(&f.pick[2], 1) & (kSelect - 1)] = u;
    });
    __syncthreads();
    const int held = c;
    const uint32_t mine = (int)threadIdx.x < held ? f.list[threadIdx.x] : kSafe;
    for (int level = 1; level < 3 && lo != hi && c != want; ++level)
      c = narrow(later, [&](auto count) {
        if ((int)threadIdx.x < held) count(mine);
      });
  }
  border = kSafe;
  take = INT32_MAX;
  if (want < 0) {  // more recent slots than the budget: the lowest
    take = budget;
  } else if (want > 0) {
    if (c != want) {  // lo == hi, and not all of the equals
      border = lo;
      take = want;
    } else if (lo == 0) {
      border = 0;
    } else {  // all from lo on
      border = lo - 1;
      take = 0;
    }
  }
}

// Keys in registers (4 Q a thread), read once.  256 heads of 16384 slots 23.6 us, of
// which reading is 9 to 10.7, the bins 6.5, the ranks 3.3, the lists 5.  They do not
// overlap: 256 heads are one workgroup a CU, and 72 registers would not let a second
// one in (seven waves a SIMD of the eight that two need).
template <int Q>
__global__ void __launch_bounds__(kSelect) evict_select_kernel(int32_t* __restrict__ holes,
                                                               int32_t* __restrict__ movers,
                                                               int32_t* __restrict__ moves,
                                                               const float* __restrict__ weight,
                                                               const int32_t* __restrict__ pos,
                                                               const int32_t* __restrict__ len,
                                                               const int32_t* __restrict__ next, int nSeq, int nHeads,
                                                               int maxSeq, int budget, int recent, int most) {
  __shared__ Search f;
  __shared__ uint32_t tab[Q * kSelectWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t head = blockIdx.x;
  const int s = (int)(head / nHeads % nSeq);
  const int n = min(max(len[s], 0), maxSeq);
  const int64_t safe = (int64_t)next[s] - recent;
  weight += head * maxSeq;
  pos += head * maxSeq;
  holes += head * most;
  movers += head * most;
  int moved = 0;
  if (n > budget) {
    uint32_t key[Q][4];
    {
      constexpr int kLoads = Q < 8 ? Q : 4;  // in flight, of both arrays
#pragma unroll
      for (int q0 = 0; q0 < Q; q0 += kLoads) {
        float w[kLoads][4];
        int p[kLoads][4];
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
          const int at = 4 * ((int)threadIdx.x + (q0 + q) * kSelect);
          if (at + 4 <= n) {
            __builtin_memcpy(w[q], weight + at, 16);
            __builtin_memcpy(p[q], pos + at, 16);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[q][e] = at + e < n ? weight[at + e] : 0.f;
              p[q][e] = at + e < n ? pos[at + e] : 0;
            }
          }
        }
#pragma unroll
        for (int q = 0; q < kLoads; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            key[q0 + q][e] = (int64_t)p[q][e] >= safe ? kSafe : weight_key(w[q][e]);
      }
    }
    auto all_keys = [&](auto use) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * ((int)threadIdx.x + q * kSelect) + e < n) use(key[q][e]);
    };
    uint32_t border;
    int take;
    find_border(all_keys, budget, f, border, take);
    int last = take == 0 ? -1 : n;  // the last slot whose key may be `border`
    // the number of flagged slots before each of a thread's, by slot order: counts
    // of (group of 4 Q, wave) summed up in a table, two flags at a time in halves of
    // 16 bits (at most 32767 slots are before one)
    uint32_t before[Q];
    auto rank_flags = [&](auto flags) {  // flags(q, e): bit 0 and bit 1
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        int mine0 = 0, mine1 = 0, all0 = 0, all1 = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int f = flags(q, e);
          const unsigned long long b0 = __ballot(f & 1), b1 = __ballot(f & 2), low = (1ull << lane) - 1;
          mine0 += __popcll(b0 & low);
          mine1 += __popcll(b1 & low);
          all0 += __popcll(b0);
          all1 += __popcll(b1);
        }
        before[q] = (uint32_t)mine0 | (uint32_t)mine1 << 16;
        if (lane == 0) tab[q * kSelectWaves + wave] = (uint32_t)all0 | (uint32_t)all1 << 16;
      }
      __syncthreads();
      if (wave == 0) {
        constexpr int each = (Q * kSelectWaves + 63) / 64;
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < each; ++i) {
          const int k = lane * each + i;
          if (k < Q * kSelectWaves) mine += tab[k];
        }
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t u = __shfl_up(upto, o, 64);
          if (lane >= o) upto += u;
        }
        upto -= mine;
#pragma unroll
        for (int i = 0; i < each; ++i) {
          const int k = lane * each + i;
          if (k < Q * kSelectWaves) {
            const uint32_t t = tab[k];
            tab[k] = upto;
            upto += t;
          }
        }
        if (lane == 63) f.pick[2] = (int)(upto & 0xFFFF);
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) before[q] += tab[q * kSelectWaves + wave];
    };
    if (take > 0 && take < INT32_MAX) {  // up to that of the equals, in slot order
      auto equal = [&](int q, int e) {
        return 4 * ((int)threadIdx.x + q * kSelect) + e < n && key[q][e] == border ? 1 : 0;
      };
      rank_flags(equal);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        int rank = (int)before[q];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (equal(q, e) && ++rank == take) f.pick[1] = 4 * ((int)threadIdx.x + q * kSelect) + e;
      }
      __syncthreads();
      last = f.pick[1];
    }
    auto place = [&](int q, int e) {  // 1: a hole, 2: a mover
      const int at = 4 * ((int)threadIdx.x + q * kSelect) + e;
      const bool kept = key[q][e] > border || (key[q][e] == border && at <= last);
      return at >= n ? 0 : at < budget ? (kept ? 0 : 1) : kept ? 2 : 0;
    };
    rank_flags(place);
    moved = f.pick[2];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      int h = (int)(before[q] & 0xFFFF), m = (int)(before[q] >> 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int f = place(q, e), at = 4 * ((int)threadIdx.x + q * kSelect) + e;
        if (f == 1 && h < most) holes[h++] = at;
        if (f == 2 && m < most) movers[m++] = at;
      }
    }
  }
  for (int i = moved + (int)threadIdx.x; i < most; i += kSelect) holes[i] = movers[i] = -1;
  if (threadIdx.x == 0) moves[head] = moved;
}

// The sum of x, two numbers in halves of 16 bits, over the workgroup's earlier
// threads; `all` gets the sum of all.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* sh, uint32_t& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 63) sh[w] = s;
  __syncthreads();
  s -= x;
  all = 0;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    const uint32_t u = sh[i];
    all += u;
    s += i < w ? u : 0;
  }
  return s;
}

// The same for heads of more slots than the registers hold: their keys are read for
// every level, then for the lists in slot order,
// four slots a thread at a time.  One head of 65536 slots 61 us, 64 heads 76, bound by
// the LDS counts and the lists' barriers (loads further ahead change nothing).
__global__ void __launch_bounds__(kSelect) evict_select_long_kernel(int32_t* __restrict__ holes,
                                                               int32_t* __restrict__ movers,
                                                               int32_t* __restrict__ moves,
                                                               const float* __restrict__ weight,
                                                               const int32_t* __restrict__ pos,
                                                               const int32_t* __restrict__ len,
                                                               const int32_t* __restrict__ next, int nSeq, int nHeads,
                                                               int maxSeq, int budget, int recent, int most) {
  __shared__ Search f;
  __shared__ uint32_t halves[kSelectWaves];
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
    auto keys = [&](uint32_t (&u)[4], int j) {
      float w[4];
      int p[4];
      if (j + 4 <= n) {
        __builtin_memcpy(w, weight + j, 16);
        __builtin_memcpy(p, pos + j, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = j + e < n ? weight[j + e] : 0.f;
          p[e] = j + e < n ? pos[j + e] : 0;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = (int64_t)p[e] >= safe ? kSafe : weight_key(w[e]);
    };
    auto all_keys = [&](auto use) {
      for (int j = 4 * (int)threadIdx.x; j < n; j += 4 * kSelect) {
        uint32_t u[4];
        keys(u, j);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < n) use(u[e]);
      }
    };
    uint32_t border;
    int take;
    find_border(all_keys, budget, f, border, take);
    int equals = 0;
    for (int j0 = 0; j0 < n; j0 += 4 * kSelect) {
      const int j = j0 + 4 * (int)threadIdx.x;
      uint32_t u[4], all, mine = 0;
      keys(u, j);
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += j + e < n && u[e] == border;
      int rank = equals + (int)sum_before(mine, halves, all);
      equals += (int)all;
      int place[4];  // 1: a hole, 2: a mover
      mine = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool kept = u[e] > border || (u[e] == border && rank < take);
        rank += u[e] == border;
        place[e] = j + e >= n ? 0 : j + e < budget ? (kept ? 0 : 1) : kept ? 2 : 0;
        mine += place[e] == 1 ? 1u : place[e] == 2 ? 0x10000u : 0u;
      }
      const uint32_t before = sum_before(mine, halves, all);
      int ih = nh + (int)(before & 0xFFFF), im = nm + (int)(before >> 16);
      nh += (int)(all & 0xFFFF);
      nm += (int)(all >> 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (place[e] == 1 && ih < most) holes[ih++] = j + e;
        if (place[e] == 2 && im < most) movers[im++] = j + e;
      }
    }
  }
  for (int i = nm + (int)threadIdx.x; i < most; i += kSelect) holes[i] = movers[i] = -1;
  if (threadIdx.x == 0) moves[head] = nm;
}

// The moves, sixteen lanes each, and the new lengths (which the selection has
// read by now).
template <int NB>
__global__ void __launch_bounds__(kThreads) kv4_move_kernel(Cache c, const int32_t* __restrict__ holes,
                                                            const int32_t* __restrict__ movers,
                                                            const int32_t* __restrict__ moves, int most, int budget) {
  const int64_t head = blockIdx.x;
  if (blockIdx.y == 0 && head < c.nSeq && threadIdx.x == 0) c.len[head] = min(slots_used(c, head), budget);
  const int n = moves[head], l = threadIdx.x & 15;
  const int64_t slot0 = head * c.maxSeq;
  uint4 *k = reinterpret_cast<uint4*>(c.k), *v = reinterpret_cast<uint4*>(c.v);
  for (int i = blockIdx.y * (kThreads / 16) + (threadIdx.x >> 4); i < n; i += gridDim.y * (kThreads / 16)) {
    const int64_t to = slot0 + holes[head * most + i], from = slot0 + movers[head * most + i];
    uint4 row;
    if (l < NB) row = k[from * NB + l];
    else if (l < 2 * NB) row = v[from * NB + l - NB];
    _Float16 a, b;
    if (l < NB) {
      a = c.kd[from * NB + l];
      b = c.vd[from * NB + l];
    }
    float w;
    int p;
    if (l == 0) {
      w = c.weight[from];
      p = c.pos[from];
    }
    if (l < NB) k[to * NB + l] = row;
    else if (l < 2 * NB) v[to * NB + l - NB] = row;
    if (l < NB) {
      c.kd[to * NB + l] = a;
      c.vd[to * NB + l] = b;
    }
    if (l == 0) {
      c.weight[to] = w;
      c.pos[to] = p;
    }
  }
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
constexpr int kMaxSlots = 1 << 30;
constexpr int kMoveParts = 65535 / FG_BEAM_STATES, kMoveGroups = 65535;  // of a fg_beam_reorder call
constexpr int kMaxHeads = 1 << 21;  // heads x sequences x layers: a workgroup of 1024 threads each
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

int check_layer(const fg_kv4_cache* c, int layer, const char* fn) {
  FG_ARG_CHECK(layer >= 0 && layer < c->nLayers, "%s: layer %d outside [0, %d)", fn, layer, c->nLayers);
  return FG_OK;
}
Cache view(const fg_kv4_cache* c, bool only_new = false) {
  return {c->nSeq,   c->nKvHeads, c->maxSeq,  c->k,      c->v,    (_Float16*)c->kd, (_Float16*)c->vd,
          c->len,    c->next,     c->weight,  c->pos,    only_new};
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

int fg::check_kv4_cache(const fg_kv4_cache* c, const char* fn) {
  FG_ARG_CHECK(c, "%s: null cache", fn);
  FG_ARG_CHECK(c->nLayers > 0 && c->nSeq > 0 && c->nKvHeads > 0 && c->maxSeq > 0,
               "%s: bad dimensions: %d layers, %d sequences, %d kv heads, %d slots", fn, c->nLayers, c->nSeq,
               c->nKvHeads, c->maxSeq);
  const int d = c->dHead;
  FG_ARG_CHECK(d == 32 || d == 64 || d == 96 || d == 128 || d == 256,
               "%s: head size %d is not one of 32, 64, 96, 128, 256", fn, d);
  FG_ARG_CHECK(c->maxSeq <= kMaxSlots, "%s: %d slots are above %d", fn, c->maxSeq, kMaxSlots);
  FG_ARG_CHECK((int64_t)c->nLayers * c->nSeq < kMaxHeads / c->nKvHeads, "%s: %d x %d x %d heads are too many", fn,
               c->nLayers, c->nSeq, c->nKvHeads);
  FG_ARG_CHECK(c->k && c->v && c->kd && c->vd && c->len && c->next, "%s: null array", fn);
  FG_ARG_CHECK(aligned16(c->k) && aligned16(c->v) && aligned16(c->kd) && aligned16(c->vd) && aligned16(c->weight) &&
                   aligned16(c->pos),
               "%s: the cache's arrays must be 16-byte aligned", fn);
  return FG_OK;
}

#define KV4_TRY(expr)                 \
  do {                                \
    const int rc_ = (expr);           \
    if (rc_ != FG_OK) return rc_;     \
  } while (0)

extern "C" int fg_kv4_append(const fg_kv4_cache* c, int layer, const float* k, const float* v, int64_t ld, int T,
                             const int32_t* count) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_append"));
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
                                   k, v, ld, T, count, (uint32_t)rows));
  return FG_OK;
}

extern "C" int fg_kv4_read(const fg_kv4_cache* c, int layer, float* k, float* v, int64_t ld, int first, int T) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_read"));
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
                                   v, ld, first, T, (uint32_t)rows));
  return FG_OK;
}

extern "C" int fg_kv4_attn(const fg_kv4_cache* c, int layer, float* out, const float* q, int nHeads, double scale,
                           int T, const int32_t* count) {
  return fg::kv4_attn(c, layer, out, q, nHeads, scale, T, count, false);
}
int fg::kv4_attn(const fg_kv4_cache* c, int layer, float* out, const float* q, int nHeads, double scale, int T,
                 const int32_t* count, bool only_new) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_attn"));
  KV4_TRY(check_layer(c, layer, "fg_kv4_attn"));
  FG_ARG_CHECK(out && q, "fg_kv4_attn: null argument");
  FG_ARG_CHECK(T >= 0, "fg_kv4_attn: T %d is negative", T);
  FG_ARG_CHECK(nHeads > 0 && nHeads % c->nKvHeads == 0, "fg_kv4_attn: %d query heads for %d kv heads", nHeads,
               c->nKvHeads);
  FG_REQUIRE_INIT();
  fg::KProfScope prof("kv4_attn", 0.0, (double)c->nSeq * c->maxSeq * slot_bytes(c));
  const int group = nHeads / c->nKvHeads, subs = (group + 7) / 8, share = (group + subs - 1) / subs;
  const int G = share > 4 ? 8 : share > 2 ? 4 : share;
  const int64_t heads = (int64_t)c->nSeq * c->nKvHeads * subs, rounds = (c->maxSeq + kRound - 1) / kRound;
  // Short caches, of more slots the more heads there are to fill the chip: a
  // workgroup a head, no second launch (but where shares of a head's query heads
  // would add to the same weights).  The host knows the slots, not how many are in
  // use.  us, a workgroup a head against pieces, every sequence full and (in
  // brackets) sequences of all lengths up to that:
  //                    up to the limit                     beyond it
  //    8 heads of 32   1536:  7.3  8.3                     2304:  9.1  8.2
  //   64 heads of 32   2048:  8.6 12.9 (2900: 10.3 12.9)   4096: 13.3 17.9 (13.2 14.0)
  //  256 heads of 32   7680: 26.5 30.8 (7600: 25.2 24.5)  11520: 37.3 38.2
  //    8 heads of 64   1280:  7.5  8.3                     1920:  9.1  8.6
  //   48 heads of 64   1280:  7.6 11.5 ( 7.4 11.2)         2048:  9.7 12.6 ( 9.7 11.6)
  //   64 heads of 64   2560: 11.2 16.0 (11.0 12.6)         4096: 15.6 20.1 (15.4 16.3)
  //  256 heads of 64   6400: 26.4 34.0 (25.6 25.3)         9600: 37.1 42.1
  //    8 heads of 96    512:  7.5  9.5  1024: 10.8  9.8    1536: 14.3 10.1
  //   64 heads of 96   2048: 17.7 19.5 (17.6 15.3)         4096: 31.1 22.9 (29.5 22.2)
  //  256 heads of 96   5120: 39.4 48.2 (37.9 35.5)         8192: 59.5 62.9
  //    8 heads of 128   896:  8.5  9.3                     1344: 10.8  9.9
  //   48 heads of 128   896:  8.5 13.0 ( 8.5 11.8)         2048: 14.3 15.2 (14.3 13.8)
  //   64 heads of 128  1792: 12.9 18.2 (12.9 14.4)         2688: 17.7 22.6 (16.9 18.6)
  //  256 heads of 128  4480: 30.0 40.2 (28.7 31.0)         8192: 55.3 64.0 (47.8 40.6)
  //    8 heads of 256   256: 10.1 11.5   384: 13.1 11.7     512: 16.0 11.8
  //   64 heads of 256   512: 16.2 16.0   768: 21.5 20.0    1152: 31.1 27.2 (1024: 26.7 18.9)
  //  256 heads of 256  1920: 55.8 61.0 (53.5 50.5)         2880: 91.8 80.2
  // Three classes of heads are coarse: from 48 to some 100 heads of 32 to 128 a
  // workgroup a head stays ahead for up to 1.5 times the limit, and heads of 96
  // and 256 cross a little before it.
  const int few = c->dHead == 32 ? 1536 : c->dHead == 64 ? 1280 : c->dHead == 96 ? 1024 : c->dHead == 128 ? 896 : 384;
  const bool whole = c->maxSeq <= few * (heads < 64 ? 1 : heads < 192 ? 2 : 5) && !(c->weight && subs > 1);
  // One sequence: equal pieces, all resident at once (130001 positions of 8 heads
  // 32.6 us, in pieces of half the size 37.4).  Several: their last pieces are
  // shorter, pieces of half the size even that out (32 sequences up to 8192
  // 40.6 us, else 47.6).
  const int cus = fg::device_cu_count() > 0 ? fg::device_cu_count() : 256;
  int target = 0;
  KV4_DISPATCH(c->dHead, target = kResident<NB> * cus);
  if (c->nSeq > 1) target *= 2;
  const int64_t grid = whole ? heads : heads * rounds < heads + target ? heads * rounds : heads + target;
  // Few heads of many pieces each are fetched by many threads (32 heads of 96
  // pieces 5.4 us, with 256 threads 9.0); others by small workgroups (1024 heads of
  // up to 11 pieces 6.4 us, with 1024 threads 12.4).
  const int kJoin = rounds > 64 && (int64_t)c->nSeq * nHeads <= 256 ? 1024 : 256;
  const int64_t chunks = c->weight ? (c->maxSeq + kJoin - 1) / kJoin : 0;
  const int64_t join = (int64_t)c->nSeq * nHeads + (int64_t)c->nSeq * c->nKvHeads * chunks;
  FG_ARG_CHECK(grid <= INT32_MAX / 512 && join <= INT32_MAX / kJoin,
               "fg_kv4_attn: %d sequences x %d heads x %d slots are too many", c->nSeq, nHeads, c->maxSeq);
  // references and sums, values, and the scores where weights are kept
  const bool pieces = !whole && (rounds > 1 || c->weight);
  const size_t ml = pieces ? (size_t)grid * G * sizeof(float2) : 0;
  const size_t po = pieces && rounds > 1 ? (size_t)grid * G * c->dHead * sizeof(float) : 0;
  const size_t ps = c->weight ? (size_t)c->nSeq * nHeads * c->maxSeq * sizeof(float) : 0;
  const Cache cache = view(c, only_new);
  fg::Workspace ws;
  if (ml + po + ps > 0) KV4_TRY(ws.get(ml + po + ps));
  float2* part_ml = (float2*)ws.ptr;
  float* part_o = (float*)((uint8_t*)ws.ptr + ml);
  float* sc = c->weight ? (float*)((uint8_t*)ws.ptr + ml + po) : nullptr;
#define KV4_ATTN(GS)                                                                                                   \
  if (whole)                                                                                                           \
    FG_LAUNCH((kv4_attn_kernel<NB, GS, true>), dim3((unsigned)grid), dim3(64 * kWholeWaves<NB, GS>), 0, cache, layer,   \
              out, q, nHeads, subs, (float)scale, T, count, target, part_ml, part_o, sc);                              \
  else                                                                                                                 \
    FG_LAUNCH((kv4_attn_kernel<NB, GS, false>), dim3((unsigned)grid), dim3(kThreads), 0, cache, layer, out, q,         \
              nHeads, subs, (float)scale, T, count, target, part_ml, part_o, sc)
#define KV4_JOIN(J)                                                                                               \
  FG_LAUNCH((kv4_join_kernel<NB, J>), dim3((unsigned)join), dim3(J), 0, cache, layer, out, nHeads, subs, G, T, count,   \
            target, (const float2*)part_ml, (const float*)part_o, (const float*)sc, (int)chunks)
  KV4_DISPATCH(c->dHead, {
    if (G == 1) {
      KV4_ATTN(1);
    } else if (G == 2) {
      KV4_ATTN(2);
    } else if (G == 4) {
      KV4_ATTN(4);
    } else {
      KV4_ATTN(8);
    }
    if (pieces) {
      if (kJoin == 1024) KV4_JOIN(1024);
      else KV4_JOIN(256);
    }
  });
#undef KV4_JOIN
#undef KV4_ATTN
  return FG_OK;
}

extern "C" int fg_kv4_commit(const fg_kv4_cache* c, int T, const int32_t* count) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_commit"));
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
  FG_ARG_CHECK(nLayers > 0 && nSeq > 0 && nHeads > 0 && maxSeq > 0 && maxSeq <= kMaxSlots &&
                   (int64_t)nLayers * nSeq < kMaxHeads / nHeads,
               "fg_kv_evict_select: bad dimensions: %d layers, %d sequences, %d heads, %d slots", nLayers, nSeq, nHeads,
               maxSeq);
  FG_ARG_CHECK(budget >= 1 && budget < maxSeq, "fg_kv_evict_select: budget %d outside [1, %d)", budget, maxSeq);
  FG_ARG_CHECK(recent >= 0 && recent <= budget, "fg_kv_evict_select: recent %d outside [0, %d]", recent, budget);
  const int heads = nLayers * nSeq * nHeads, most = budget < maxSeq - budget ? budget : maxSeq - budget;
  FG_REQUIRE_INIT();
  fg::KProfScope prof("kv_evict_select", 0.0, (double)heads * (8.0 * maxSeq + 8.0 * most));
  // Keys in registers up to 32768 slots: 128 heads of 32768 35.2 us, read from memory
  // for every level 42.2; 256 of 16384 23.6 and 26.2.  At 65536 they would not fit:
  // 64 heads 76 us from memory, 91 from registers that spill.
#define EVICT_SELECT(kernel)                                                                                    \
  FG_LAUNCH((kernel), dim3(heads), dim3(kSelect), 0, holes, movers, moves, weight, pos, len, next, nSeq, nHeads, \
            maxSeq, budget, recent, most)
  if (maxSeq <= 4 * kSelect) EVICT_SELECT(evict_select_kernel<1>);
  else if (maxSeq <= 8 * kSelect) EVICT_SELECT(evict_select_kernel<2>);
  else if (maxSeq <= 16 * kSelect) EVICT_SELECT(evict_select_kernel<4>);
  else if (maxSeq <= 32 * kSelect) EVICT_SELECT(evict_select_kernel<8>);
  else EVICT_SELECT(evict_select_long_kernel);
#undef EVICT_SELECT
  return FG_OK;
}

extern "C" int fg_kv4_evict(const fg_kv4_cache* c, int budget, int recent) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_evict"));
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
  const int want = (most + kThreads / 16 - 1) / (kThreads / 16), fit = (4096 + heads - 1) / heads;
  const dim3 grid(heads, want < fit ? want : fit);
  KV4_DISPATCH(c->dHead, FG_LAUNCH(kv4_move_kernel<NB>, grid, dim3(kThreads), 0, view(c), (const int32_t*)holes,
                                   (const int32_t*)movers, (const int32_t*)moves, most, budget));
  return FG_OK;
}

extern "C" int fg_kv4_reorder(const fg_kv4_cache* c, const int32_t* parent, int W) {
  KV4_TRY(fg::check_kv4_cache(c, "fg_kv4_reorder"));
  FG_ARG_CHECK(parent, "fg_kv4_reorder: null argument");
  FG_ARG_CHECK(W >= 1 && W <= 64 && c->nSeq % W == 0, "fg_kv4_reorder: %d sequences are not groups of %d beams "
               "(1 to 64)", c->nSeq, W);
  FG_REQUIRE_INIT();
  // a launch takes so many parts (layers x kv heads) and requests: larger caches go in
  // several, the lengths read by all of them and moved at the end
  const int heads = c->nKvHeads < kMoveParts ? c->nKvHeads : kMoveParts, layers = kMoveParts / heads;
  const int groups = c->nSeq / W;
  for (int r0 = 0; r0 < groups; r0 += kMoveGroups)
    for (int l0 = 0; l0 < c->nLayers; l0 += layers)
      for (int h0 = 0; h0 < c->nKvHeads; h0 += heads) {
        fg_beam_state st[6];
        int n = 0;
        auto add = [&](void* base, int64_t row) {
          if (!base) return;
          const int64_t head = c->maxSeq * row, seq = c->nKvHeads * head, layer = c->nSeq * seq;
          st[n++] = {(uint8_t*)base + l0 * layer + (int64_t)r0 * W * seq + h0 * head, seq,
                     min(layers, c->nLayers - l0), layer, min(heads, c->nKvHeads - h0), head, row, c->maxSeq};
        };
        add(c->k, c->dHead / 2);
        add(c->v, c->dHead / 2);
        add(c->kd, c->dHead / 16);
        add(c->vd, c->dHead / 16);
        add(c->weight, 4);
        add(c->pos, 4);
        const int64_t at = (int64_t)r0 * W;
        KV4_TRY(fg_beam_reorder(st, n, parent + at, c->len + at, min(kMoveGroups, groups - r0), W));
      }
  FG_LAUNCH(kv4_follow_kernel, dim3(c->nSeq / W), dim3(64), 0, c->len, c->next, parent, W);
  return FG_OK;
}
