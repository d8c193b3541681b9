// WindowAttention for many rows: prompts, pieces of prompts, image patches.
//
// The products are fp32 and the matrix instruction for fp32 does 152 TFLOP/s on a large product;
// those for 16-bit operands do 1100.  An fp32 operand is therefore taken as a sum of two fp16 numbers,
// x * 2^e = hi + lo, each rounded to nearest: 22 bits of it, and a product as
//   hi hi' + hi lo' + lo hi'
// of three, accumulated in fp32 (lo lo' is 2^-22 of it and left out).  That is within a factor of
// what fp32 operands leave, at twice to three times their rate.  The powers of two keep operands in
// fp16's range: one for a row of q, one for a tile of keys, one for a tile of values.
//
// attention_split_kernel splits the keys and values that any query sees once, in tiles of 32 keys,
// into the order in which the lanes of v_mfma_f32_32x32x16_f16 take them: a workgroup copies
// a tile to LDS as it lies there and reads it as it lies there.  Keys and values are used by a workgroup for
// every 128 rows, so splitting them where they are used would cost as much as the weights' exponentials.
//
// attention_tiles_kernel: scores come out as S^T (keys x rows), a row in two lanes; 16 weights of a
// lane, rounded to hi and lo, are the operand of the second product as they are, since its
// contraction may take the keys in any order and the values are stored in that order.
//
// A tile is left to the fp32 instruction, from the caches themselves, where a power of two for the whole tile or row
// would cost precision: where that shows in the scores (loss), where its values' rows and columns differ in size (value_factor),
// where values in front of it were far smaller than its own (rough_values), or where something in it is not
// finite.  So a row that does not see (or hardly weighs) an outlier, and a column that has none, does not suffer from it.
//
// A causal prompt of 4096 tokens, 32 heads of 128 values on 8: 370 us, 137 GFLOP of products or 1.11 PFLOP/s of fp16 ones, what
// a large library product reaches; the split is 13 us of it.  577 patches that all see each other, 16 images, 12 heads of 64: 95 us,
// the split 21 (113 MB), rows in and out 12, of the rest a half products.  Pieces of 999 tokens in a window of 512, 12 heads of 80:
// 53 us, 288 workgroups on 256 compute units, so that some have two.  4096 tokens, 16 heads on 4 of 256: 491, of 160 or 192 values
// (both have room for 192) 350.  A prompt whose tiles all need fp32 takes ten times as long as one that needs none.
#include "attention_common.h"

#include "../../include/shadow_hip.h"
#include "attention_tiles.h"
#include "launch.h"
#include "split16.h"

#include <type_traits>

#pragma clang fp contract(off)

namespace shdw {

constexpr int kTile = 32;         // keys
constexpr int kWaveRows = 32;

struct alignas(16) TileInfo {
  float key_factor;    // 2^-e of the keys
  float key_sum;       // the largest sum of |x| of a key
  float value_factor;  // 2^-e of the values; NaN: they need fp32 operands, infinite: and so does all behind them
  float value_least;   // the largest |value| of the row that has the smallest one, rows of zeros apart
};

// The tiles of 32 keys, counted from key 0, that queries between two reaches see: [0, sinks) and [lo, hi).
struct TileSpan {
  int sinks, lo, hi;
};
SHDW_DEVICE TileSpan span_of(const Reach& a, const Reach& b) {
  TileSpan s;
  s.sinks = (b.first + kTile - 1) / kTile;
  s.lo = max(a.lo / kTile, s.sinks);
  s.hi = max((b.hi + kTile - 1) / kTile, s.lo);
  return s;
}

constexpr int kMostLift = 30;  // of values, either way

// A workgroup a tile, eight lanes a key, everything read once: keys stay in registers while the largest
// values are found, values go through LDS, from where they are taken value by value.
template <int NB>
__global__ __launch_bounds__(kBlock) void attention_split_kernel(const float* k, const float* v, v8h* parts, TileInfo* infos,
                                                                  FastDiv f_tiles, AttentionArgs p) {
  constexpr int kPadded = 32 * NB, kChunks = kPadded / 8, kEach = (kChunks + 7) / 8;  // chunks of 8 values, of a lane
  __shared__ float most[2][kBlock / kWave], other[2][kBlock / kWave], columns[2][kPadded];  // other: sums of keys, the least values
  __shared__ v4f rows[kTile][kPadded / 4 + 1];  // keys start in other banks
  const int tid = threadIdx.x;
  uint32_t head, slot;
  fd_divmod(blockIdx.x, f_tiles, head, slot);
  const uint32_t b = fd_div(head, p.f_kv);
  const Sequence seq = sequence_of(p, b);
  if (seq.count == 0) return;
  const Reach first = reach_of(p, seq, 0), last = reach_of(p, seq, seq.count - 1);
  const TileSpan span = span_of(first, last);
  const int tile = static_cast<int>(slot) < span.sinks ? static_cast<int>(slot) : span.lo + static_cast<int>(slot) - span.sinks;
  if (tile >= span.hi && tile >= span.sinks) return;
  const int key = tid / 8, part = tid % 8, j = tile * kTile + key;
  const bool live = j < last.first || (j >= first.lo && j < last.hi);  // what no query sees counts as zeros
  const uint64_t row = (static_cast<uint64_t>(head) * p.capacity + j) * p.dim;

  float x[2][kEach][8];
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int c = 0; c < kEach; ++c) {
      const int d = 8 * (part + 8 * c);
      const float* from = (which ? v : k) + row + d;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[which][c][i] = 0.f;
      if (live && d < p.dim) {
        if (d + 8 <= p.dim) {
          const v4f e = load4_any(from), f = load4_any(from + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[which][c][i] = e[i], x[which][c][4 + i] = f[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (d + i < p.dim) x[which][c][i] = from[i];
        }
      }
    }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float m = 0.f, sum = 0.f;
#pragma unroll
    for (int c = 0; c < kEach; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m = larger_or_nan(m, __builtin_fabsf(x[which][c][i]));
        if (which == 0) sum += __builtin_fabsf(x[which][c][i]);
      }
    m = larger_or_nan(m, dpp_f32<kDppXor1>(m));
    m = larger_or_nan(m, dpp_f32<kDppXor2>(m));
    m = larger_or_nan(m, dpp_f32<kDppHalfMirror>(m));
    if (which == 0) {
      sum += dpp_f32<kDppXor1>(sum);
      sum += dpp_f32<kDppXor2>(sum);
      sum += dpp_f32<kDppHalfMirror>(sum);
    } else {
      sum = m == 0.f ? -INFINITY : -m;
    }
    for (int step = 8; step < kWave; step <<= 1) {
      m = larger_or_nan(m, __shfl_xor(m, step));
      const float next = __shfl_xor(sum, step);
      sum = which == 0 ? larger_or_nan(sum, next) : larger(sum, next);
    }
    if (tid % kWave == 0) most[which][tid / kWave] = m, other[which][tid / kWave] = sum;
  }
#pragma unroll
  for (int c = 0; c < kEach; ++c)
    if (part + 8 * c < kChunks) {
      rows[key][2 * (part + 8 * c)] = v4f{x[1][c][0], x[1][c][1], x[1][c][2], x[1][c][3]};
      rows[key][2 * (part + 8 * c) + 1] = v4f{x[1][c][4], x[1][c][5], x[1][c][6], x[1][c][7]};
    }
  __syncthreads();
  float largest[2] = {most[0][0], most[1][0]}, key_sum = other[0][0], smallest = -other[1][0];
#pragma unroll
  for (int w = 1; w < kBlock / kWave; ++w) {
    largest[0] = larger_or_nan(largest[0], most[0][w]), largest[1] = larger_or_nan(largest[1], most[1][w]);
    key_sum = larger_or_nan(key_sum, other[0][w]);
    smallest = __builtin_fminf(smallest, -other[1][w]);
  }
  const int key_lift = lift_of(largest[0]);
  // Steps of 2^4, so that neighbouring tiles mostly agree: the largest in [2^10, 2^14).  In tiles that are not whole the
  // smallest column may be a single small number: they have the most bits that there are.
  const bool part_of_tile = !((tile + 1) * kTile <= last.first || (tile * kTile >= first.lo && (tile + 1) * kTile <= last.hi));
  const int value_lift = largest[1] == 0.f ? kMostLift : part_of_tile ? 13 - exponent_of(largest[1]) : 10 - (exponent_of(largest[1]) & ~3);
  // sums in units of these could leave fp32's range; 128 is what the exponent of infinities and NaN gives
  const bool wild_values = value_lift > kMostLift || value_lift < -kMostLift;
  if (tid == 0) {
    infos[blockIdx.x].key_factor = power2(-key_lift), infos[blockIdx.x].key_sum = key_sum;
    infos[blockIdx.x].value_least = smallest;
    if (wild_values) infos[blockIdx.x].value_factor = value_lift < 0 ? INFINITY : NAN;
  }

  // [keys hi][keys lo][values hi][values lo], each 32 * kPadded numbers
  constexpr uint32_t kQuarter = kTile * kPadded / 8;
  v8h* out = parts + static_cast<uint64_t>(blockIdx.x) * 4 * kQuarter;
#pragma unroll
  for (int c = 0; c < kEach; ++c) {
    const int chunk = part + 8 * c;
    if (chunk >= kChunks) break;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[0][c][i] *= power2(key_lift);
    v8h hi, lo;
    split8(x[0][c], hi, lo);
    const uint32_t at = (chunk / 2) * kWave + (chunk % 2) * 32 + key;
    out[at] = hi;
    out[kQuarter + at] = lo;
  }
  if (wild_values) return;
  const float* const values = reinterpret_cast<const float*>(rows);
#pragma unroll
  for (int n = tid; n < 4 * kPadded; n += kBlock) {
    // value d of keys 16 m + 8 a + 4 h + t, element 4 a + t
    const int d = n / 128 * 32 + n % 32, h = n / 32 % 2, m = n / 64 % 2;
    float w[8], column = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = values[(16 * m + 8 * (i / 4) + 4 * h + i % 4) * (kPadded + 4) + d];
      column = larger(column, __builtin_fabsf(w[i]));
      w[i] *= power2(value_lift);
    }
    column = across_halves(column, larger);  // of keys 16 m ..
    if (h == 0) columns[m][d] = column;
    v8h hi, lo;
    split8(w, hi, lo);
    out[2 * kQuarter + n] = hi;
    out[3 * kQuarter + n] = lo;
  }
  // Where rows and columns differ in size, values of a small row in a small column are about (smallest row) (smallest column) /
  // largest.  What the second part of a number rounds away is up to 2^-25 in units of the lift; it has to be less
  // than 2^-21 of those.
  __syncthreads();
  if (tid >= kWave) return;
  float column = INFINITY;
  for (int d = tid; d < kPadded; d += kWave) {
    const float c = larger(columns[0][d], columns[1][d]);
    if (c > 0.f) column = __builtin_fminf(column, c);
  }
  for (int step = 1; step < kWave; step <<= 1) column = __builtin_fminf(column, __shfl_xor(column, step));
  if (tid == 0) {
    const float factor = power2(-value_lift), small = smallest / largest[1] * column;
    infos[blockIdx.x].value_factor = largest[1] == 0.f || factor <= 16.f * small ? factor : NAN;
  }
}

// Copies one tile to LDS, every wave its share, 16 bytes a lane and turn.
template <int BYTES, int WAVES>
SHDW_DEVICE void fetch(const char* from, char* to, int wave, int lane) {
  constexpr int kTurns = BYTES / (WAVES * kWave * 16);
#pragma unroll
  for (int n = 0; n < kTurns; ++n) {
    const int at = (wave * kTurns + n) * kWave * 16;
    to_lds16(from + at + lane * 16, to + at);
  }
}

// The weights that go to the second product are 2^(score - top + 12): at most 2^15 while `top` lags behind
// by up to kLag, and down to 2^-37 of the largest before fp16 rounds them away.  What is rounded away counts as its values do:
// a tile whose values are up to 2^12 times the smallest row's in front of it adds 2^-25 of these for a key at most, others have fp32
// weights.
constexpr float kLift = 12.f, kLag = 3.f;

// The tiles that go through fp32 operands are rare and their code is long: functions of their own, so that the
// others' registers do not depend on them.
// Scores of a tile, a lane's key and row given, as the kernel for few rows has them.
template <int NB>
__device__ __attribute__((noinline)) v16f fp32_scores(const float* key, const float* row, int dim, float scale) {
  const int half = threadIdx.x % kWave / 32;
  v16f s = {};
#pragma unroll 1
  for (int c = 0; c < 2 * NB; ++c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 16 * c + 8 * half + e;
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(d < dim ? key[d] : 0.f, d < dim ? row[d] * scale : 0.f, s, 0, 0, 0);
    }
  }
  return s;
}
// `sum` and up to 32 dims of the tile's values from key j0 on, weighted.  Values that are not finite count as zeros; a row that
// sees one becomes NaN.
__device__ __attribute__((noinline)) v16f fp32_values(const float* values, int dim, int dims, int j0, int keys, Reach reach, v16f weights,
                                                      v16f sum) {
  const int lane = threadIdx.x % kWave, half = lane / 32, i = lane % 32;
  bool hurt = false;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = j0 + 8 * (r / 4) + 4 * half + r % 4;
    float x = j < keys && i < dims ? values[static_cast<uint64_t>(j) * dim + i] : 0.f;
    const bool off = !(__builtin_fabsf(x) < INFINITY);
    x = off ? 0.f : x;
    sum = __builtin_amdgcn_mfma_f32_32x32x2f32(x, weights[r], sum, 0, 0, 0);
    const uint64_t votes = __builtin_amdgcn_ballot_w64(off);
    hurt = hurt || (static_cast<uint32_t>(votes >> (32 * half)) != 0 && sees(reach, j));
  }
  const float bad = across_halves(hurt ? 1.f : 0.f, larger) != 0.f ? NAN : 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) sum[r] += bad;
  return sum;
}

// A wave has 32 rows.  Tiles are copied to LDS up to BUFFERS - 1 ahead of their use.
template <int NB, int WAVES, int BUFFERS>
__global__ __launch_bounds__(WAVES * kWave, NB <= 4 ? 2 : 1) void attention_tiles_kernel(
    const float* q, const float* k, const float* v, float* y, const v8h* parts, const TileInfo* infos, float* sums,
    uint32_t tiles, FastDiv f_heads, FastDiv f_splits, uint32_t blocks, AttentionArgs p) {
  constexpr int kPadded = 32 * NB, kBytes = 4 * kTile * kPadded * 2, kAhead = BUFFERS - 1, kTileRows = kWaveRows * WAVES;
  __shared__ alignas(16) char lds[BUFFERS][kBytes];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32, i = lane % 32;
  // the last rows of a causal prompt have the most keys: they go first
  const uint32_t splits = f_splits.d;
  uint32_t rest, head, part, block, b, h;
  fd_divmod(blockIdx.x, f_heads, rest, head);
  fd_divmod(rest, f_splits, block, part);
  fd_divmod(head, p.f_kv, b, h);
  block = blocks - 1 - block;
  const int base = block * kTileRows, row = base + kWaveRows * wave + i;
  uint32_t t, shared;
  fd_divmod(min(row, p.length * p.group - 1), p.f_group, t, shared);
  const bool quads = p.dim % 4 == 0;
  const uint64_t at = ((static_cast<uint64_t>(b) * p.length + t) * p.q_heads + h * p.group + shared) * p.dim;

  // the row: dims 16 s + 8 half + e.  Asked for before anything that has to be waited for; values behind the last dim are
  // made 0 below.
  float x[2 * NB][8];
  if (quads) {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const v4f w = load4_any(q + at + min(16 * s + 8 * half + e, p.dim - 4));
#pragma unroll
        for (int c = 0; c < 4; ++c) x[s][e + c] = w[c];
      }
  } else {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = q[at + min(16 * s + 8 * half + e, p.dim - 1)];
  }
  asm volatile("" ::: "memory");

  const Sequence seq = sequence_of(p, b);
  const int rows = seq.count * p.group;
  if (base >= rows) return;
  const auto query_reach = [&](int row) { return reach_of(p, seq, fd_div(min(row, rows - 1), p.f_group)); };
  const TileSpan whole = span_of(reach_of(p, seq, 0), reach_of(p, seq, seq.count - 1));
  const TileSpan span = span_of(query_reach(base), query_reach(base + kTileRows - 1));
  const Reach wave_a = query_reach(base + 32 * wave), wave_b = query_reach(base + 32 * wave + 31);
  const Reach reach = reach_of(p, seq, min(static_cast<int>(t), seq.count - 1));
  const bool mine = row < rows;
  const uint64_t cache = static_cast<uint64_t>(head) * p.capacity * p.dim;
  const char* tile_parts = reinterpret_cast<const char*>(parts) + static_cast<uint64_t>(head) * tiles * kBytes;

  const int count = span.sinks + span.hi - span.lo;
  int from, to;
  part_of(count, part, f_splits, from, to);
  const auto tile_at = [&](int n) { return n < span.sinks ? n : span.lo + n - span.sinks; };
  const auto slot_at = [&](int tile) { return tile < whole.sinks ? tile : tile - whole.lo + whole.sinks; };
  // A tile's info comes by scalar loads, which are counted apart from the copies that are under way.
  typedef const __attribute__((address_space(4))) TileInfo* InfoPointer;
  const InfoPointer tile_infos = reinterpret_cast<InfoPointer>(reinterpret_cast<uintptr_t>(infos + static_cast<uint64_t>(head) * tiles));
  const auto info_at = [&](int n) {
    const InfoPointer at = tile_infos + slot_at(tile_at(n));
    TileInfo info;
    info.key_factor = at->key_factor, info.value_factor = at->value_factor;
    info.value_least = at->value_least, info.key_sum = at->key_sum;
    return info;
  };
  // What all tiles of the part have in common, a lane a tile: asked for here, in front of the copies.
  uint32_t most_factor = 0, least_value = __float_as_uint(INFINITY);  // positive numbers compare like their bits
  float key_sum = 0.f, key_factor = 0.f;
  for (int n = from + lane; n < to; n += kWave) {
    const TileInfo info = infos[static_cast<uint64_t>(head) * tiles + slot_at(tile_at(n))];
    key_sum = larger_or_nan(key_sum, info.key_sum), key_factor = larger(key_factor, info.key_factor);
    most_factor = max(most_factor, __float_as_uint(info.value_factor));
    least_value = min(least_value, __float_as_uint(info.value_least));
  }
  const auto ask = [&](int n, int buffer) {
    if (n < to) fetch<kBytes, WAVES>(tile_parts + static_cast<uint64_t>(slot_at(tile_at(n))) * kBytes, lds[buffer], wave, lane);
  };
  if (from < to) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) ask(from + a, a);
  }

  v8h qhi[2 * NB], qlo[2 * NB];
  float row_factor, wave_most, wave_sum;  // of the wave's rows
  {
    float m = 0.f, sum = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = 16 * s + 8 * half + e < p.dim ? x[s][e] * (p.scale * kLog2e) : 0.f;
        m = larger(m, __builtin_fabsf(x[s][e]));
        sum += __builtin_fabsf(x[s][e]);
      }
    m = across_halves(m, larger), sum = across_halves(sum, plus);
    wave_most = mine ? m : 0.f, wave_sum = mine ? sum : 0.f;
    for (int step = 1; step < 32; step <<= 1) {
      wave_most = larger(wave_most, __shfl_xor(wave_most, step));
      wave_sum = larger(wave_sum, __shfl_xor(wave_sum, step));
    }
    wave_most = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(wave_most)));
    wave_sum = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(wave_sum)));
    const int e = lift_of(m);
    const float f = power2(e);
    row_factor = power2(-e);
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) {
#pragma unroll
      for (int c = 0; c < 8; ++c) x[s][c] *= f;
      split8(x[s], qhi[s], qlo[s]);
    }
  }

  v16f acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[n][r] = 0.f;
  float top = -INFINITY, total = 0.f, unit = 1.f;  // acc is in units of `unit`, a tile's value_factor

  // What the second parts of keys and rows round away, up to 2^-38 of a row's and of a tile's largest number, adds up to this in a
  // score, every rounding at its worst (a twentieth of it is what is met).  It has to stay below 2^-20, or below 2^-22 of the row's
  // largest score, where fp32 sums are no better: else, and where something is not finite, the tile's scores are fp32 products.
  const auto loss = [&](float sum, float factor) { return (wave_most * sum + wave_sum * (factor * 0x1p14f)) * 0x1p-38f; };
  // Values of a tile, less than 2^14 times their factor, are up to 2^12 times the least row's, or need fp32 weights; so does a
  // factor that is a NaN.
  const auto rough_weights = [](uint32_t factor, uint32_t least) { return factor + (2u << 23) > least; };
  for (int step = 1; step < kWave; step <<= 1) least_value = min(least_value, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least_value), step)));
  // Mostly nothing is rough: a loop that does not ask.  Asking in every tile a prompt of 4096 takes 400 us for 370, heads of 256
  // twice as long, since the calls want registers.
  const bool smooth = __builtin_amdgcn_ballot_w64(!(loss(key_sum, key_factor) <= 0x1p-20f) || rough_weights(most_factor, least_value)) == 0;
  int buffer = 0;
  uint32_t least = __float_as_uint(INFINITY);  // of the tiles so far, in a scalar register
  bool far = false;                            // sums may be too large to be taken to other units
  const auto all = [&](auto ask_each) {
    constexpr bool kAsk = decltype(ask_each)::value;
    for (int n = from; n < to; ++n) {
      const int tile = tile_at(n), j0 = tile * kTile;
      const char* here = lds[buffer];
      const TileInfo info = info_at(n);  // in front of the wait: reads of LDS behind it are then counted alone
      // the tile is there (later ones may be under way), and nobody reads the buffer that is filled next
      if (to - n >= kAhead) copies_done<(kAhead - 1) * kBytes / (WAVES * kWave * 16)>();
      else copies_done<0>();
      ask(n + kAhead, buffer == 0 ? BUFFERS - 1 : buffer - 1);
      buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
      // a tile that none of the wave's rows sees
      if (!(j0 < wave_b.first || (j0 < wave_b.hi && j0 + kTile > wave_a.lo))) continue;

      v16f s;
      float f, m;
      const auto score = [&](bool fp32) {
        if (!fp32) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 0.f;
          const v8h* frag = reinterpret_cast<const v8h*>(here) + lane;
#pragma unroll
          for (int c = 0; c < 2 * NB; ++c) {
            const v8h hi = frag[c * kWave], lo = frag[(2 * NB + c) * kWave];
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, qhi[c], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, qlo[c], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, qhi[c], s, 0, 0, 0);
          }
          f = __builtin_fmaxf(__builtin_fminf(row_factor * info.key_factor, 0x1p127f), 0x1p-126f);  // neither 0 nor infinite
        } else {
          s = fp32_scores<NB>(k + cache + static_cast<uint64_t>(min(j0 + i, p.capacity - 1)) * p.dim, q + at, p.dim, p.scale * kLog2e);
          f = 1.f;
          loads_done();
        }
        if (!((j0 + kTile <= wave_a.first) || (j0 >= wave_b.lo && j0 + kTile <= wave_a.hi))) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!sees(reach, j0 + 8 * (r / 4) + 4 * half + r % 4)) s[r] = -INFINITY;
        }
        m = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) m = larger(m, s[r]);
        m = across_halves(m, larger);
        m = m == -INFINITY ? m : m * f;
      };
      if constexpr (kAsk) {
        const float lost = loss(info.key_sum, info.key_factor);
        const auto rough = [&] { return __builtin_amdgcn_ballot_w64(mine && lost > 0x1p-22f * larger(4.f, __builtin_fabsf(m))) != 0; };
        bool fp32 = !(lost < INFINITY);
        if constexpr (NB != 4) {  // of 4 that spills registers: such tiles among others 891 us for a prompt of 4096, 494 in a loop
          if (!fp32) {
            score(false);
            fp32 = rough();
          }
          if (fp32) score(true);
        } else {
          for (;; fp32 = true) {
            score(fp32);
            if (fp32 || !rough()) break;
          }
        }
      } else {
        score(false);
      }
      least = min(least, __float_as_uint(info.value_least));
      far = kAsk && (far || info.value_factor == INFINITY);
      const bool rough_values = kAsk && (far || rough_weights(__float_as_uint(info.value_factor), least));
      if (__builtin_amdgcn_ballot_w64(m > (rough_values ? top : top + kLag)) != 0) {
        const float next = larger(m, top);
        const float g = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
        top = next;
        total *= g;
#pragma unroll
        for (int b2 = 0; b2 < NB; ++b2)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[b2][r] *= g;
      }
      // Scores of 2^22 and more have steps of a half and more: rounded as `top` is they are at most top + kLag, in one step they could
      // be far above it, and their weights infinite in fp16.  Where nothing is lost they are below 2^18.
      const float base = top == -INFINITY ? 0.f : top, shift = base - kLift;
      float part_sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(kAsk ? (s[r] * f - base) + kLift : __builtin_fmaf(s[r], f, -shift));
        part_sum += s[r];
      }
      total += part_sum;

      if (!rough_values) {
        if (info.value_factor != unit) {
          const float g = unit * (1.f / info.value_factor);  // powers of two
          unit = info.value_factor;
#pragma unroll
          for (int b2 = 0; b2 < NB; ++b2)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[b2][r] *= g;
        }
        v8h whi[2], wlo[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float w[8] = {s[8 * c], s[8 * c + 1], s[8 * c + 2], s[8 * c + 3], s[8 * c + 4], s[8 * c + 5], s[8 * c + 6], s[8 * c + 7]};
          split8(w, whi[c], wlo[c]);
        }
        const v8h* frag = reinterpret_cast<const v8h*>(here) + 4 * NB * kWave + lane;
#pragma unroll
        for (int b2 = 0; b2 < NB; ++b2)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const v8h hi = frag[(2 * b2 + c) * kWave], lo = frag[(2 * NB + 2 * b2 + c) * kWave];
            acc[b2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, whi[c], acc[b2], 0, 0, 0);
            acc[b2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, wlo[c], acc[b2], 0, 0, 0);
            acc[b2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, whi[c], acc[b2], 0, 0, 0);
          }
      } else {
        // weights of up to 1, as the kernel for few rows has them: nothing overflows here that does not there
        const float g = unit * __builtin_exp2f(-kLift);
        unit = __builtin_exp2f(kLift);
#pragma unroll
        for (int b2 = 0; b2 < NB; ++b2)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[b2][r] *= g;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= __builtin_exp2f(-kLift);
#pragma unroll
        for (int b2 = 0; b2 < NB; ++b2)
          acc[b2] = fp32_values(v + cache + 32 * b2, p.dim, p.dim - 32 * b2, j0, seq.keys, reach, s, acc[b2]);
        loads_done();
      }
    }
  };
  if (__builtin_expect(smooth, 1)) all(std::false_type());
  else all(std::true_type());
  if (!mine) return;
  total = across_halves(total, plus);
  if (WAVES == 8 || splits == 1) {
    const bool empty = sees_nothing(reach);
    const float g = unit / total;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v4f o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = empty ? 0.f : acc[n][4 * c + e] * g;
        const int d = 32 * n + 8 * c + 4 * half;
        if (d + 4 <= p.dim) {
          *reinterpret_cast<v4f_unaligned*>(y + at + d) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < p.dim) y[at + d + e] = o[e];
        }
      }
  } else {
    const uint64_t slot = ((static_cast<uint64_t>(head) * blocks + block) * splits + part) * kTileRows + 32 * wave + i;
    const uint64_t slots = static_cast<uint64_t>(gridDim.x) * kTileRows;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v4f o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = acc[n][4 * c + e] * (unit * __builtin_exp2f(-kLift));
        *reinterpret_cast<v4f*>(sums + slot * kPadded + 32 * n + 8 * c + 4 * half) = o;
      }
    if (half == 0) {
      sums[slots * kPadded + 2 * slot] = top;
      sums[slots * kPadded + 2 * slot + 1] = total * __builtin_exp2f(-kLift);
    }
  }
}

bool plan_tiles(int batch, int length, int q_heads, int kv_heads, int dim, int capacity, int window, int sinks, int causal,
                TilesPlan* plan) {
  const int64_t rows = static_cast<int64_t>(length) * (q_heads / kv_heads), heads = static_cast<int64_t>(batch) * kv_heads;
  const int n = (dim + 31) / 32;
  plan->padded = 32 * (n == 5 ? 6 : n == 7 ? 8 : n);
  // Heads of 128 values: eight waves share a tile of 32 KB where rows fill the chip with them twice over (a causal prompt of
  // 4096 for 32 heads 370 us against 393 with four), four have less to wait for where they do not (pieces of 999 in a
  // window of 512 66 against 87).  Shorter heads: four (64 values, 577 patches of 16 images 95 against 121).
  plan->waves = plan->padded == 128 && (rows + 255) / 256 * heads >= 512 ? 8 : 4;
  const uint32_t block_rows = kWaveRows * plan->waves;
  const int64_t blocks = (rows + block_rows - 1) / block_rows, items = blocks * heads;
  int64_t tiles = (static_cast<int64_t>(capacity) + kTile - 1) / kTile;
  if (window > 0)
    tiles = std::min<int64_t>(tiles, (static_cast<int64_t>(sinks) + kTile - 1) / kTile +
                                         (static_cast<int64_t>(window) * (causal ? 1 : 2) + length) / kTile + 2);
  tiles = std::max<int64_t>(tiles, 1);
  // parts of the keys, where rows alone do not fill the chip: none with fewer than eight tiles.  Two workgroups for a compute unit:
  // with one 1000 tokens of 32 heads take 62.8 us (60.5), 16 sequences with 96 rows over 1900 keys 52.3 (50.6); with four the first
  // 68.1, pieces of 999 in a window of 512 79 (66), and 96 rows over 4000 keys of 8 heads gain 0.3 of 37.6
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / items, tiles / 8, 64}));
  if (!grid_fits(items * splits, plan->waves * kWave) || !grid_fits(heads * tiles, kBlock)) return false;
  plan->blocks = static_cast<uint32_t>(blocks), plan->splits = static_cast<uint32_t>(splits);
  plan->tiles = static_cast<uint32_t>(tiles), plan->heads = static_cast<uint32_t>(heads);
  plan->parts_bytes = static_cast<size_t>(heads * tiles) * 4 * kTile * plan->padded * 2;
  plan->infos_bytes = static_cast<size_t>(heads * tiles) * sizeof(TileInfo);
  plan->sums_bytes = splits == 1 ? 0 : static_cast<size_t>(items * splits) * block_rows * (plan->padded + 2) * sizeof(float);
  return true;
}

template <int NB, int WAVES, int BUFFERS>
static int launch_tiles_of(const TilesPlan& plan, const float* q, const float* k, const float* v, float* y, void* workspace,
                           const AttentionArgs& p, hipStream_t st) {
  char* at = static_cast<char*>(workspace);
  v8h* parts = reinterpret_cast<v8h*>(at);
  TileInfo* infos = reinterpret_cast<TileInfo*>(at + plan.parts_bytes);
  float* sums = reinterpret_cast<float*>(at + plan.parts_bytes + plan.infos_bytes);
  attention_split_kernel<NB><<<plan.heads * plan.tiles, kBlock, 0, st>>>(k, v, parts, infos, make_fastdiv(plan.tiles), p);
  if (int rc = launch_status()) return rc;
  attention_tiles_kernel<NB, WAVES, BUFFERS><<<plan.heads * plan.blocks * plan.splits, WAVES * kWave, 0, st>>>(
      q, k, v, y, parts, infos, sums, plan.tiles, make_fastdiv(plan.heads), make_fastdiv(plan.splits), plan.blocks, p);
  if (int rc = launch_status()) return rc;
  if (plan.splits == 1) return SHDW_OK;
  static_assert(WAVES == 4 || WAVES == 8, "eight waves, whose workgroups fill the chip, have one part");
  return join_parts(sums, y, plan.splits, plan.blocks, 7, plan.padded, plan.heads, p, st);
}

int launch_tiles(const TilesPlan& plan, const float* q, const float* k, const float* v, float* y, void* workspace,
                 const AttentionArgs& p, hipStream_t st) {
  switch (plan.padded / 32) {
    case 1: return launch_tiles_of<1, 4, 2>(plan, q, k, v, y, workspace, p, st);
    case 2: return launch_tiles_of<2, 4, 2>(plan, q, k, v, y, workspace, p, st);
    case 3: return launch_tiles_of<3, 4, 2>(plan, q, k, v, y, workspace, p, st);
    case 4:
      return plan.waves == 8 ? launch_tiles_of<4, 8, 4>(plan, q, k, v, y, workspace, p, st)
                             : launch_tiles_of<4, 4, 2>(plan, q, k, v, y, workspace, p, st);
    case 6: return launch_tiles_of<6, 4, 3>(plan, q, k, v, y, workspace, p, st);
    default: return launch_tiles_of<8, 4, 2>(plan, q, k, v, y, workspace, p, st);
  }
}

}  // namespace shdw
