// Connected4: y [rows][out] = x [rows][in] W^T + bias with weights of four bits,
//   W[o][k] = low[o][k / group] + step[o][k / group] * code[o][k],  code in 0..15.
// Eight codes stand in a 32-bit word, code k in bits 4 (k % 8) of word k / 8; in is a multiple of
// 8.  Without `lows` a group's low end is -8 steps.  The reference's fully connected operator has
// fp32 weights only.
//
// A group's part of an output is step * sum(code * x) + low * sum(x), the sums on matrix instructions, the rest in fp32.  Both
// sums are in units of a power of two that x is scaled by, which is undone behind the step: in x's own units they would leave
// fp32's range from |x| of 2^117 on, where x and the result are still within it.
//
// Up to 8 rows: the codes are read once and that is the time, and unpacking them what stands in its way.  x becomes
// a whole number of 23 bits and a sign in units of a group's power of two, in three digits to the base 256; four rows' digits are
// the 16 rows of the int8 instruction (one of four is not used), codes are int8 numbers after three instructions for
// eight, and sums are exact.  Workgroups take 16 or 32 outputs, their eight waves an eighth of `in` each.  Digits of one row
// every workgroup makes for itself, of more rows a launch of their own does (2.6 us).  4096 x 6144 weights for one row 6.9 us
// (1.9 TB/s of codes and steps), 4096 x 32000 17.0 (4.1 TB/s), 4096 x 16384 with low ends for four rows 13.6 (3.1 TB/s): what is left
// is launches, the first loads and the steps, which every output has to itself.
//
// More rows, by 16: the same with x split into two fp16 numbers, 22 bits of it, since three digits would
// be three times the products to scale; 5000 x 4099 weights for 13 rows 14.9 us, of which x, read by every workgroup, is most, 16384 x 4096 with
// low ends for 16 rows 17.2, for 64 49.1.  A code as fp16: four bits at the bottom of 0x6400 are 1024 + code, in the next
// four bits 1024 + 16 code, so one AND-OR and one packed subtraction make two operands out of a word (nibbles 0 and 4,
// 1 and 5, and 2 and 6, 3 and 7 after one shift); the odd nibbles' x is a sixteenth.  (The bits alone are the
// subnormal code * 2^-24, which the instruction takes, but adds up with an error of 5 10^-6: it aligns products by the
// exponents of the factors.)
//
// From 80 to some hundred rows on, the fewer the larger the weights: x is split once into the order in which lanes take it, tiles of
// 128 rows x 128 outputs copy it to LDS,
// four waves of 64 x 64 unpack the codes in registers.  700 rows on 4096 x 4096 weights 84 us, 560 TFLOP/s of fp16 products: 192
// tiles are a workgroup for three of four compute units, and LDS, unpacking and products take turns there.  Tiles of 64 rows
// 86.6, eight waves of 32 x 32 102.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/shadow_hip.h"
#include "device_common.h"
#include "launch.h"
#include "split16.h"

#pragma clang fp contract(off)

namespace shdw {

struct Connected4Args {
  uint32_t rows, words, out, groups;
  const float* steps;
  const float* lows;
  const float* bias;
};

// The operand of one word: nibbles 0 4 1 5 2 6 3 7, the odd ones 16 times as large.
SHDW_DEVICE v8h operand_of(uint32_t word) {
  const uint32_t high = word >> 8;
  uint32_t k1024 = 0x64006400u;
  asm("" : "+v"(k1024));  // two constants are two instructions, a constant and a register one
  const v4u bits = {(word & 0x000f000fu) | k1024, (word & 0x00f000f0u) | k1024, (high & 0x000f000fu) | k1024,
                    (high & 0x00f000f0u) | k1024};
  return __builtin_bit_cast(v8h, bits) - static_cast<_Float16>(1024.f);
}
// Eight values of x, lifted, in the same order, split.
SHDW_DEVICE void operand_of(const float (&x)[8], v8h& hi, v8h& lo) {
  constexpr int kNibble[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = kNibble[e] % 2 ? x[kNibble[e]] * 0.0625f : x[kNibble[e]];
  split8(v, hi, lo);
}
SHDW_DEVICE void load8(const float* p, float (&x)[8]) {
  const v4f a = load4_any(p), b = load4_any(p + 4);
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] = a[c], x[4 + c] = b[c];
}
SHDW_DEVICE v4u load_words(const uint32_t* p) {  // at any dword address
  typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(4)));
  return *reinterpret_cast<const v4u_any*>(p);
}
template <int LANES, class F>
SHDW_DEVICE float across_lanes(float v, F&& join) {  // groups of 4, 8 or 16 lanes
  v = join(v, dpp_f32<kDppXor1>(v));
  v = join(v, dpp_f32<kDppXor2>(v));
  if (LANES >= 8) v = join(v, dpp_f32<kDppHalfMirror>(v));
  if (LANES >= 16) v = join(v, dpp_f32<kDppMirror>(v));
  return v;
}
SHDW_DEVICE void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
SHDW_DEVICE void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8;
constexpr int kBlockWords = 16;            // 128 codes: 16 bytes a lane and output
constexpr uint32_t kFewFloats = 12288;     // steps of a workgroup's outputs and factors of x that LDS holds at a time
constexpr uint32_t kFewBlockBytes = 2048;  // of a set of four rows: 16 operand rows of 128 digits

typedef int v4i __attribute__((ext_vector_type(4)));

// The register that a word of a block is in, and its lane group, once words of one group of x are in one register
// (groups of 32 codes), in two (64) or as they were loaded (128).
template <int GROUP_WORDS>
SHDW_DEVICE void few_place(int word, int& g, int& t) {
  if (GROUP_WORDS == 16) {
    g = word / 4, t = word % 4;
  } else if (GROUP_WORDS == 8) {
    g = (word / 2 % 2) * 2 + word / 4 % 2, t = word / 8 * 2 + word % 2;
  } else {
    g = word % 4, t = word / 4;
  }
}

// A lane's word of a row as digits, and its group's factor that undoes the power of two and sum, in units of the last digit
// (times -8 without lows).
struct Digits {
  uint2 top, middle, low;  // eight digits each: of even codes, of odd ones
  float factor, sum;
};
template <int GROUP_WORDS, bool LOWS>
SHDW_DEVICE Digits digits_of(const float (&v)[8]) {
  float most = 0.f, sum = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c) most = larger_or_nan(most, __builtin_fabsf(v[c]));
  most = across_lanes<GROUP_WORDS>(most, [](float a, float b) { return larger_or_nan(a, b); });
  // the largest in [2^22, 2^23) / 1.0045: three digits hold up to 127 * 65793 = 2^23 / 1.0039; up to 2^149, with which
  // subnormal numbers are whole
  const int e = 22 - exponent_of(most * 1.0045f);
  uint32_t top[2] = {}, middle[2] = {}, low[2] = {};
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    // v = 65536 a + 256 b + c, each in -128 .. 127
    const float scaled = lifted(v[c], e);
    sum += scaled;
    const int d = static_cast<int>(__builtin_rintf(scaled));
    const int lo = static_cast<int8_t>(d), rest = (d - lo) >> 8, mid = static_cast<int8_t>(rest), hi = (rest - mid) >> 8;
    const int word = c % 2, byte = c / 2 * 8;  // even codes in one register, odd ones in the next
    top[word] |= static_cast<uint32_t>(hi & 255) << byte;
    middle[word] |= static_cast<uint32_t>(mid & 255) << byte;
    low[word] |= static_cast<uint32_t>(lo & 255) << byte;
  }
  Digits d;
  d.top = make_uint2(top[0], top[1]), d.middle = make_uint2(middle[0], middle[1]), d.low = make_uint2(low[0], low[1]);
  d.factor = most < INFINITY ? lift_undone(e) : NAN;  // digits hold nothing that is not finite
  sum = across_lanes<GROUP_WORDS>(sum, [](float a, float b) { return a + b; });
  d.sum = LOWS ? sum : sum * -8.f;
  return d;
}

// Digits of x: [set][block][two registers][lane group][4 rows x 4 digits][register][8], and [group][set][row][factor, sum].
// A lane a word of a row.
template <int GROUP_WORDS, bool LOWS>
__global__ __launch_bounds__(kBlock) void connected4_digits_kernel(const float* x, char* digits, float* factors, uint32_t words,
                                                                   uint32_t blocks, uint32_t sets) {
  const uint32_t row = blockIdx.y, set = row / 4, at = blockIdx.x * kBlock + threadIdx.x, block = at / kBlockWords;
  if (block >= blocks) return;  // whole groups of lanes
  float v[8];
  if (at < words) {
    load8(x + (static_cast<uint64_t>(row) * words + at) * 8, v);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = 0.f;
  }
  const Digits d = digits_of<GROUP_WORDS, LOWS>(v);
  int g, t;
  few_place<GROUP_WORDS>(at % kBlockWords, g, t);
  char* to = digits + (static_cast<uint64_t>(set) * blocks + block) * kFewBlockBytes + (t / 2) * 1024 + g * 256 + row % 4 * 64 + t % 2 * 8;
  *reinterpret_cast<uint2*>(to) = d.top;
  *reinterpret_cast<uint2*>(to + 16) = d.middle;
  *reinterpret_cast<uint2*>(to + 32) = d.low;
  if (at % GROUP_WORDS == 0) {
    float* out = factors + ((static_cast<uint64_t>(at / GROUP_WORDS) * sets + set) * 4 + row % 4) * 2;
    out[0] = d.factor, out[1] = d.sum;
  }
}

// Adds to `sum` the products of a block with the digits x0, x1; factors: of the block's first group, PITCH floats a group.
template <int GROUP_WORDS, bool LOWS, int PITCH>
SHDW_DEVICE void add_digits(v4u x0, v4u x1, const v4u (&b)[2], const float* factors, const float* step, const float* low, float& sum) {
  const v4i zero = {0, 0, 0, 0};
  const auto add = [&](int u, v4i d) {
    const float2 factor = *reinterpret_cast<const float2*>(factors + u * PITCH);
    const float f = __builtin_fmaf(static_cast<float>(d[0]), 65536.f, __builtin_fmaf(static_cast<float>(d[1]), 256.f, static_cast<float>(d[2])));
    sum = __builtin_fmaf(LOWS ? __builtin_fmaf(factor.y, low[u], f * step[u]) : (f + factor.y) * step[u], factor.x, sum);
  };
  const v4u x[2] = {x0, x1};
  if (GROUP_WORDS == 4) {
    constexpr int kLast = kBlockWords / GROUP_WORDS - 1;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint64_t a = static_cast<uint64_t>(x[t / 2][t % 2 * 2 + 1]) << 32 | x[t / 2][t % 2 * 2];
      const uint64_t c = static_cast<uint64_t>(b[t / 2][t % 2 * 2 + 1]) << 32 | b[t / 2][t % 2 * 2];
      add(min(t, kLast), __builtin_amdgcn_mfma_i32_16x16x32_i8(static_cast<long>(a), static_cast<long>(c), zero, 0, 0, 0));
    }
  } else {
    constexpr int kLast = GROUP_WORDS == 8 ? 1 : 0;
    const v4i one = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, x0), __builtin_bit_cast(v4i, b[0]), zero, 0, 0, 0);
    if (GROUP_WORDS == 8) add(0, one);
    add(kLast, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, x1), __builtin_bit_cast(v4i, b[1]),
                                                     GROUP_WORDS == 8 ? zero : one, 0, 0, 0));
  }
}
SHDW_DEVICE void codes_as_int8(const uint32_t (&w)[4], v4u (&b)[2]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) b[t / 2][t % 2 * 2] = w[t] & 0x0f0f0f0fu, b[t / 2][t % 2 * 2 + 1] = w[t] >> 4 & 0x0f0f0f0fu;
}

// One row: every workgroup makes the digits itself, into LDS, 512 bytes a block; the operand's other rows are this one
// once more.
template <int GROUP_WORDS, bool LOWS>
struct OneRow {
  static constexpr bool kOwn = true;
  static constexpr int kGroups = kBlockWords / GROUP_WORDS, kRows = 1, kSums = 1, kLoads = 0, kFactors = 2, kFloats = 128;
  struct Operands {};
  int lane;
  SHDW_DEVICE OneRow(const char*, uint32_t, uint32_t, int l) : lane(l / 16 * 4 + l % 4) {}
  SHDW_DEVICE void load(uint32_t, Operands&) const {}
  // Digits of word `at` of the chunk, which is word c of x.
  static SHDW_DEVICE void put(const float (&v)[8], uint32_t at, float* digits, float* factors) {
    const Digits d = digits_of<GROUP_WORDS, LOWS>(v);
    int g, t;
    few_place<GROUP_WORDS>(at % kBlockWords, g, t);
    char* to = reinterpret_cast<char*>(digits + at / kBlockWords * kFloats) + (t / 2) * 256 + g * 64 + t % 2 * 8;
    *reinterpret_cast<uint2*>(to) = d.top;
    *reinterpret_cast<uint2*>(to + 16) = d.middle;
    *reinterpret_cast<uint2*>(to + 32) = d.low;
    if (at % GROUP_WORDS == 0) factors[at / GROUP_WORDS * 2] = d.factor, factors[at / GROUP_WORDS * 2 + 1] = d.sum;
  }
  SHDW_DEVICE void multiply(const Operands&, const float* digits, const float* factors, int, const uint32_t (&w)[4],
                            const float (&step)[kGroups], const float (&low)[kGroups], float (&sums)[kSums]) const {
    v4u b[2];
    codes_as_int8(w, b);
    const v4u* x = reinterpret_cast<const v4u*>(digits) + lane;
    add_digits<GROUP_WORDS, LOWS, kFactors>(x[0], x[16], b, factors, step, low, sums[0]);
  }
  static SHDW_DEVICE uint32_t row(int, int g) { return g; }  // only one is there
};

// x of up to 8 rows as digits: SETS sets of four rows, a lane's sum of set s is row 4 s + lane / 16.
template <int GROUP_WORDS, int SETS, bool LOWS>
struct DigitRows {
  static constexpr bool kOwn = false;
  static constexpr int kFloats = 0, kGroups = kBlockWords / GROUP_WORDS, kRows = 4 * SETS, kSums = SETS, kLoads = 2 * SETS, kFactors = 8 * SETS;
  struct Operands {
    v4u x[SETS][2];
  };
  const char* digits;
  uint32_t blocks;
  int lane;
  SHDW_DEVICE DigitRows(const char* parts, uint32_t all_blocks, uint32_t, int l) : digits(parts), blocks(all_blocks), lane(l) {}
  SHDW_DEVICE void load(uint32_t block, Operands& k) const {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const char* from = digits + (static_cast<uint64_t>(s) * blocks + block) * kFewBlockBytes + lane * 16;
      k.x[s][0] = *reinterpret_cast<const v4u*>(from);
      k.x[s][1] = *reinterpret_cast<const v4u*>(from + 1024);
    }
  }
  SHDW_DEVICE void multiply(const Operands& k, const float*, const float* factors, int g, const uint32_t (&w)[4],
                            const float (&step)[kGroups], const float (&low)[kGroups], float (&sums)[kSums]) const {
    v4u b[2];
    codes_as_int8(w, b);
#pragma unroll
    for (int s = 0; s < SETS; ++s)
      add_digits<GROUP_WORDS, LOWS, kFactors>(k.x[s][0], k.x[s][1], b, factors + s * 8 + g * 2, step, low, sums[s]);
  }
  static SHDW_DEVICE uint32_t row(int sum, int g) { return 4 * sum + g; }
};

// x of up to 16 rows as two fp16 numbers: [block][register][lane group][row][hi, lo], [group][16] factors and [16]
// sums, in the products' units.  A lane's sums are rows 4 (lane / 16) ..
template <int GROUP_WORDS, bool LOWS>
__global__ __launch_bounds__(kBlock) void connected4_halves_kernel(const float* x, char* parts, float* factors, uint32_t words,
                                                                   uint32_t blocks) {
  const uint32_t row = blockIdx.y % 16, set = blockIdx.y / 16, at = blockIdx.x * kBlock + threadIdx.x, block = at / kBlockWords;
  if (block >= blocks) return;  // whole groups of lanes
  float v[8];
  if (at < words) {
    load8(x + (static_cast<uint64_t>(blockIdx.y) * words + at) * 8, v);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = 0.f;
  }
  float most = 0.f, sum = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c) most = larger(most, __builtin_fabsf(v[c]));
  most = across_lanes<GROUP_WORDS>(most, [](float a, float b) { return larger(a, b); });
  const int e = far_lift_of(most);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    v[c] = lifted(v[c], e);
    sum += v[c];
  }
  sum = across_lanes<GROUP_WORDS>(sum, [](float a, float b) { return a + b; });
  v8h hi, lo;
  operand_of(v, hi, lo);
  int g, t;
  few_place<GROUP_WORDS>(at % kBlockWords, g, t);
  v8h* to = reinterpret_cast<v8h*>(parts + ((((static_cast<uint64_t>(set) * blocks + block) * 4 + t) * 4 + g) * 16 + row) * 32);
  to[0] = hi, to[1] = lo;
  if (at % GROUP_WORDS == 0) {
    const uint64_t groups = static_cast<uint64_t>(blocks) * (kBlockWords / GROUP_WORDS);
    float* out = factors + (set * groups + at / GROUP_WORDS) * 32 + row;
    out[0] = lift_undone(e), out[16] = LOWS ? sum : sum * -8.f;
  }
}
template <int GROUP_WORDS, bool LOWS>
struct HalfRows {
  static constexpr bool kOwn = false;
  static constexpr int kFloats = 0, kGroups = kBlockWords / GROUP_WORDS, kRows = 16, kSums = 4, kLoads = 8, kFactors = 32;
  struct Operands {
    v8h hi[4], lo[4];
  };
  const char* parts;
  SHDW_DEVICE HalfRows(const char* from, uint32_t, uint32_t rows, int lane)
      : parts(from + (lane / 16 * 16 + min(static_cast<uint32_t>(lane % 16), rows - 1)) * 32) {}  // rows that are not there: the last
  SHDW_DEVICE void load(uint32_t block, Operands& k) const {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const v8h* at = reinterpret_cast<const v8h*>(parts + (static_cast<uint64_t>(block) * 4 + t) * 4 * 16 * 32);
      k.hi[t] = at[0], k.lo[t] = at[1];
    }
  }
  SHDW_DEVICE void multiply(const Operands& k, const float*, const float* factors, int g, const uint32_t (&w)[4],
                            const float (&step)[kGroups], const float (&low)[kGroups], float (&sums)[kSums]) const {
    v4f part, sum;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const v8h b = operand_of(w[t]);
      if (t % (GROUP_WORDS / 4) == 0) {
        sum = *reinterpret_cast<const v4f*>(factors + t / (GROUP_WORDS / 4) * kFactors + 16 + 4 * g);
        part = LOWS ? v4f{0.f, 0.f, 0.f, 0.f} : sum;
      }
      part = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.hi[t], b, part, 0, 0, 0);
      part = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.lo[t], b, part, 0, 0, 0);
      if ((t + 1) % (GROUP_WORDS / 4) == 0) {
        const int u = t / (GROUP_WORDS / 4);
        const v4f undo = *reinterpret_cast<const v4f*>(factors + u * kFactors + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sums[r] = __builtin_fmaf(LOWS ? __builtin_fmaf(sum[r], low[u], part[r] * step[u]) : part[r] * step[u], undo[r], sums[r]);
      }
    }
  }
  static SHDW_DEVICE uint32_t row(int sum, int g) { return 4 * g + sum; }
};

// A workgroup: TILES tiles of 16 outputs, all of `in` for one set of rows.
template <class ROWS, int GROUP_WORDS, int TILES, bool LOWS>
__global__ __launch_bounds__(kFewWaves * kWave) void connected4_few_kernel(const float* x, const char* parts, const float* factors,
                                                                           const uint32_t* codes, float* y, uint32_t blocks,
                                                                           uint32_t chunk_blocks, size_t set_parts,
                                                                           size_t set_factors, Connected4Args p) {
  extern __shared__ v4f lds4[];
  float* const digits = reinterpret_cast<float*>(lds4);                                      // [block][kFloats]
  float* const group_factors = digits + chunk_blocks * ROWS::kFloats;                        // [group of the chunk][kFactors]
  float* const group_steps = group_factors + chunk_blocks * ROWS::kGroups * ROWS::kFactors;  // [16 TILES][pitch], then the lows
  constexpr int kGroups = ROWS::kGroups;                     // of a block
  // Blocks under way: four where they are small, else one, which leaves registers for a second workgroup (13 rows 13.5 us with
  // one, 15.2 with two, 20.7 with three; 8 rows on 16384 x 4096 16.2 and 17.1).
  constexpr int kAhead = TILES + ROWS::kLoads <= 4 ? 4 : 1;
  constexpr int kTurn = 4;  // 16384 outputs for four rows 14.7 us, 15.0 with two, 14.5 with eight, where 13 rows spill (18.5 for 15.1)
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), g = lane / 16, j = lane % 16;
  const uint32_t first_out = blockIdx.x * TILES * 16, first_row = blockIdx.y * ROWS::kRows;
  const ROWS rows(ROWS::kOwn ? nullptr : parts + blockIdx.y * set_parts, blocks, min(p.rows - first_row, 16u), lane);

  // offsets of a lane behind what the workgroup has in common
  const uint32_t* const wg_codes = codes + static_cast<uint64_t>(first_out) * p.words;
  const float* const wg_steps = p.steps + static_cast<uint64_t>(first_out) * p.groups;
  const float* const wg_lows = LOWS ? p.lows + static_cast<uint64_t>(first_out) * p.groups : nullptr;
  uint32_t local[TILES];
#pragma unroll
  for (int n = 0; n < TILES; ++n) local[n] = min(static_cast<uint32_t>(n * 16 + j), p.out - 1 - first_out);

  struct Block {
    v4u codes[TILES];
    typename ROWS::Operands x;
  };
  const auto load = [&](uint32_t block, Block& k) {
#pragma unroll
    for (int n = 0; n < TILES; ++n) k.codes[n] = load_words(wg_codes + block * kBlockWords + (local[n] * p.words + 4 * g));
    rows.load(block, k.x);
  };
  // the last block where it is not whole: x is 0 behind its end
  const auto load_tail = [&](uint32_t block, Block& k) {
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) k.codes[n][c] = wg_codes[local[n] * p.words + min(block * kBlockWords + 4 * g + c, p.words - 1)];
    rows.load(block, k.x);
  };

  float sums[TILES][ROWS::kSums] = {};
  const uint32_t pitch = chunk_blocks * kGroups | 1;
  const float* const my_steps = group_steps + j * pitch;
  const float* const my_lows = my_steps + TILES * 16 * pitch;
  const auto work = [&](const Block& k, uint32_t at) {  // `at`: block of the chunk
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      float step[kGroups], low[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        step[u] = my_steps[n * 16 * pitch + at * kGroups + u];
        low[u] = LOWS ? my_lows[n * 16 * pitch + at * kGroups + u] : 0.f;
      }
      uint32_t w[4] = {k.codes[n][0], k.codes[n][1], k.codes[n][2], k.codes[n][3]};
      if (GROUP_WORDS <= 8) swap32(w[0], w[2]), swap32(w[1], w[3]);
      if (GROUP_WORDS == 4) swap16(w[0], w[1]), swap16(w[2], w[3]);
      rows.multiply(k.x, digits + at * ROWS::kFloats, group_factors + at * kGroups * ROWS::kFactors, g, w, step, low, sums[n]);
    }
  };

  // the workgroup's steps go through LDS: a lane's own would be sixteen lines for every four or eight bytes, which costs
  // more than the codes
  for (uint32_t chunk = 0; chunk < blocks; chunk += chunk_blocks) {
    const uint32_t here = min(chunk_blocks, blocks - chunk), whole = min(p.words / kBlockWords, chunk + here) - chunk;
    const uint32_t from = chunk + whole * wave / kFewWaves, to = chunk + whole * (wave + 1) / kFewWaves;
    const uint32_t first_group = chunk * kGroups, columns = here * kGroups;
    // a wave's share of the steps: turns of 64 groups of every eighth output, kTurn turns on their way at once
    struct Turns {
      float step[kTurn], low[kTurn];
      uint32_t at[kTurn];
    };
    uint32_t turn_row = wave, turn_column = 0;
    const auto ask = [&](Turns& t) {
#pragma unroll
      for (int u = 0; u < kTurn; ++u) {
        const uint32_t row = min(turn_row, TILES * 16u - 1), column = turn_column + lane;
        const uint64_t from_row = static_cast<uint64_t>(min(row, p.out - 1 - first_out)) * p.groups;
        const uint32_t group = min(first_group + column, p.groups - 1);
        t.step[u] = (wg_steps + from_row)[group];
        if (LOWS) t.low[u] = (wg_lows + from_row)[group];
        t.at[u] = turn_row < TILES * 16 && column < columns ? row * pitch + column : ~0u;
        turn_column += kWave;
        if (turn_column >= columns) turn_column = 0, turn_row += kFewWaves;
      }
    };
    const auto put = [&](const Turns& t) {
#pragma unroll
      for (int u = 0; u < kTurn; ++u)
        if (t.at[u] != ~0u) {
          group_steps[t.at[u]] = t.step[u];
          if (LOWS) group_steps[t.at[u] + TILES * 16 * pitch] = t.low[u];
        }
    };
    Turns turns;
    ask(turns);
    const v4f* from_factors = reinterpret_cast<const v4f*>(factors + blockIdx.y * set_factors + static_cast<uint64_t>(first_group) * ROWS::kFactors);
    const uint32_t quads = ROWS::kOwn ? 0 : columns * (ROWS::kFactors / 4);
    v4f some[2];
    float own[8];
    const auto ask_own = [&](uint32_t at) { load8(x + 8ull * min(chunk * kBlockWords + at, p.words - 1), own); };
    if constexpr (ROWS::kOwn) {
      ask_own(threadIdx.x);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) some[u] = from_factors[min(threadIdx.x + u * kFewWaves * kWave, quads - 1)];
    }
    asm volatile("" ::: "memory");
    Block k[kAhead];
    if (from < to) {
      // every load is made, the ones behind the end once more: a load that may not be made would have to be
      // waited for as if it were the last
#pragma unroll
      for (int a = 0; a < kAhead; ++a) load(min(from + a, to - 1), k[a]);
    }
    asm volatile("" ::: "memory");
    if (chunk > 0) __syncthreads();
    put(turns);
    if constexpr (ROWS::kOwn) {
      for (uint32_t at = threadIdx.x;;) {  // whole groups of lanes
        if (at >= here * kBlockWords) break;
        if (chunk * kBlockWords + at >= p.words) {
#pragma unroll
          for (int c = 0; c < 8; ++c) own[c] = 0.f;
        }
        ROWS::put(own, at, digits, group_factors);
        at += kFewWaves * kWave;
        ask_own(at);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (threadIdx.x + u * kFewWaves * kWave < quads) lds4[threadIdx.x + u * kFewWaves * kWave] = some[u];
    while (turn_row < TILES * 16) {
      ask(turns);
      asm volatile("" ::: "memory");
      put(turns);
    }
    for (uint32_t c = threadIdx.x + 2 * kFewWaves * kWave; c < quads; c += kFewWaves * kWave) lds4[c] = from_factors[c];
    __syncthreads();  // also keeps the loads of codes in front of it, not where their values are first used
    if (from < to)
      for (uint32_t block = from;; block += kAhead) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (block + a < to) work(k[a], block + a - chunk);
        if (block + kAhead >= to) break;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) load(min(block + kAhead + a, to - 1), k[a]);
        asm volatile("" ::: "memory");  // the loads go out here
      }
    if (whole < here && wave == kFewWaves - 1) {
      load_tail(chunk + whole, k[0]);
      work(k[0], whole);
    }
  }

  __syncthreads();
  float* const share = reinterpret_cast<float*>(lds4);  // nobody reads steps any more
#pragma unroll
  for (int n = 0; n < TILES; ++n)
#pragma unroll
    for (int i = 0; i < ROWS::kSums; ++i) share[((wave * TILES + n) * ROWS::kSums + i) * kWave + lane] = sums[n][i];
  __syncthreads();
  constexpr int kAll = TILES * ROWS::kSums;
  for (int at = wave; at < kAll; at += kFewWaves) {
    float sum = share[at * kWave + lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) sum += share[(w * kAll + at) * kWave + lane];
    const uint32_t o = first_out + at / ROWS::kSums * 16 + j, row = first_row + ROWS::row(at % ROWS::kSums, g);
    if (o < p.out && row < p.rows) y[static_cast<uint64_t>(row) * p.out + o] = p.bias ? sum + p.bias[o] : sum;
  }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
constexpr int kManyRows = 128, kManyOut = 128;  // of a workgroup
constexpr int kStageWords = 8;                  // 64 codes
constexpr uint32_t kStageBytes = 2 * 32 * kStageWords * 16;  // of 32 rows: hi, lo
constexpr int kStageSums = 128;                 // of 32 rows: sums and factors of two groups
constexpr int kSplitRows = 8, kSplitParts = 4;

// Words of a stage in the order of the four products: words 0 1 4 5 in lanes 0..31, 2 3 6 7 in lanes 32..63.
SHDW_DEVICE int stage_lane(int word, int row) { return (word & 2) * 16 + row; }
SHDW_DEVICE int stage_product(int word) { return (word >> 2) * 2 + (word & 1); }

// x in the order that the lanes of the products take it: [32 rows][stage][hi, lo][product][lane], and of every
// stage and row the sums over groups that start there, [32 rows][stage][2][32], and behind these, [2][32], what takes a group's
// products to the row's units.  A workgroup takes eight rows and a part of `in`, after the largest value of the rows, which gives
// their power of two.  A group whose largest value is less than 2^-8 of the row's has a power of its own, undone before its
// steps: in the row's it would be held to 2^-34 of the row's largest value (odd codes' numbers are 2^4 smaller), which shows where
// that one meets small weights.  Other groups share the row's and need no factor; `apart`, a word for every
// workgroup, says whether any has its own.
constexpr float kNear = 0x1p-8f;
constexpr int kMostLift = 120;  // of a group above its row: 2^-kMostLift is normal
template <int GROUP_WORDS, bool LOWS>
__global__ __launch_bounds__(kBlock) void connected4_split_kernel(const float* x, v8h* parts, float* sums, float* undo, uint32_t* apart,
                                                                  uint32_t rows, uint32_t words, uint32_t stages) {
  const int lane = threadIdx.x % 32, sub = threadIdx.x / 32;  // 32 lanes a row
  const uint32_t row = blockIdx.x * kSplitRows + sub;
  const bool there = row < rows;
  const float* xr = x + static_cast<uint64_t>(min(row, rows - 1)) * words * 8;
  float most = 0.f;
  // four loads on their way at once, here and below: one at a time is 10.2 us for 700 rows of 4096, four 8.1
  constexpr int kTurns = 4;
  for (uint32_t w = lane; w < words; w += 32 * kTurns) {
    float v[kTurns][8];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) load8(xr + 8ull * min(w + 32 * n, words - 1), v[n]);
#pragma unroll
    for (int n = 0; n < kTurns; ++n)
#pragma unroll
      for (int c = 0; c < 8; ++c) most = larger(most, __builtin_fabsf(v[n][c]));
  }
  for (int s = 1; s < 32; s <<= 1) most = larger(most, __shfl_xor(most, s));
  const int e = far_lift_of(most);
  if (blockIdx.y == 0 && lane == 0) undo[row] = lift_undone(e);
  const uint32_t turns = (stages + 3) / 4;  // of 32 words: four stages, whole groups
  const uint32_t from = turns * blockIdx.y / kSplitParts, to = turns * (blockIdx.y + 1) / kSplitParts;
  const uint32_t block = row / 32, r = row % 32;
  bool own = false;
  for (uint32_t turn = from; turn < to; turn += kTurns) {
    float all[kTurns][8];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) load8(xr + 8ull * min((turn + n) * 32 + lane, words - 1), all[n]);
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      const uint32_t w = (turn + n) * 32 + lane, stage = w / kStageWords;
      if (turn + n >= to) break;
      const bool real = there && w < words;
      float v[8], group_most = 0.f, sum = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = real ? all[n][c] : 0.f;
        group_most = larger(group_most, __builtin_fabsf(v[c]));
      }
      group_most = across_lanes<GROUP_WORDS>(group_most, [](float a, float b) { return larger(a, b); });
      const int lift = group_most == 0.f || group_most >= most * kNear ? e : min(far_lift_of(group_most), e + kMostLift);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] *= power2(min(e, 126));
      if (e > 126) {  // rare, like the next: branches, not multiplications for all
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] *= power2(e - 126);
      }
      // in the units of the products, where they are added to them, else in the row's
#pragma unroll
      for (int c = 0; c < 8; ++c) sum += v[c];
      if (lift != e) {
        float own_sum = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          v[c] = lifted(real ? all[n][c] : 0.f, lift);
          own_sum += v[c];
        }
        if (!LOWS) sum = own_sum;
        own = true;
      }
      sum = across_lanes<GROUP_WORDS>(sum, [](float a, float b) { return a + b; });
      if (stage >= stages) continue;
      const int word = w % kStageWords;
      v8h hi, lo;
      operand_of(v, hi, lo);
      v8h* out = parts + (static_cast<uint64_t>(block) * stages + stage) * (kStageBytes / 16) + stage_product(word) * kWave +
                 stage_lane(word, r);
      out[0] = hi;
      out[kStageBytes / 32] = lo;
      float* const group = sums + (static_cast<uint64_t>(block) * stages + stage) * kStageSums + word / 4 * 32 + r;
      if (w % GROUP_WORDS == 0) group[0] = LOWS ? sum : sum * -8.f;
      if (w % min(GROUP_WORDS, kStageWords) == 0) group[64] = power2(e - lift);
    }
  }
  const int any = __syncthreads_or(own);
  if (threadIdx.x == 0) apart[blockIdx.x * kSplitParts + blockIdx.y] = any;
}

// What a workgroup has of a stage in LDS, all of it copied there without a register in between: x and its sums of
// four blocks of 32 rows; codes, steps and lows of four blocks of 32 outputs.
struct alignas(16) ManyStage {
  char x[4][kStageBytes];
  float sums[4][kStageSums];
  v4u codes[4][32][2];  // [output][half a row]
  float steps[4][64], lows[4][64];  // [group of the stage][output]
};
constexpr int kManyBuffers = 3;

// p[0] and p[64], and four each from p, p + 8, p + 16 and p + 24 on, of what was copied to LDS.  Read by instructions of our own,
// waited for at once: in front of a read that it sees to alias such a copy the compiler waits for all copies that are under
// way, two stages of them.
SHDW_DEVICE uint32_t lds_address(const float* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const float*)p));
}
SHDW_DEVICE v2f lds_pair(const float* p) {
  v2f v;
  asm volatile("ds_read2_b32 %0, %1 offset0:0 offset1:64\n\ts_waitcnt lgkmcnt(0)" : "=v"(v) : "v"(lds_address(p)) : "memory");
  return v;
}
SHDW_DEVICE v16f lds_rows(const float* p) {
  v4f a, b, c, d;
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:32\n\tds_read_b128 %2, %4 offset:64\n\t"
               "ds_read_b128 %3, %4 offset:96\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d) : "v"(lds_address(p)) : "memory");
  return v16f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], c[0], c[1], c[2], c[3], d[0], d[1], d[2], d[3]};
}

template <int GROUP_WORDS, bool LOWS>
__global__ __launch_bounds__(kBlock, 1) void connected4_many_kernel(const v8h* parts, const float* sums, const float* undo,
                                                                    const uint32_t* apart, const uint32_t* codes, float* y, float* partial,
                                                                    uint32_t stages, uint32_t splits, uint32_t row_tiles,
                                                                    Connected4Args p) {
  __shared__ ManyStage lds[kManyBuffers];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32, j = lane % 32;
  const uint32_t row_tile = blockIdx.x % row_tiles, part = blockIdx.x / row_tiles % splits, out_tile = blockIdx.x / row_tiles / splits;
  const int wave_rows = wave % 2, wave_out = wave / 2;  // 64 each
  const uint32_t from = static_cast<uint32_t>(static_cast<uint64_t>(stages / 2) * part / splits) * 2;
  const uint32_t to = part + 1 == splits ? stages : static_cast<uint32_t>(static_cast<uint64_t>(stages / 2) * (part + 1) / splits) * 2;

  // a wave copies block `wave` of the rows and of the outputs
  const uint32_t first_out = out_tile * kManyOut + wave * 32;
  const uint64_t my_codes = static_cast<uint64_t>(min(first_out + lane / 2, p.out - 1)) * p.words;
  const uint64_t my_groups = static_cast<uint64_t>(min(first_out + lane % 32, p.out - 1)) * p.groups;
  const char* const my_x = reinterpret_cast<const char*>(parts) + static_cast<uint64_t>(row_tile * 4 + wave) * stages * kStageBytes + lane * 16;
  const float* const my_sums = sums + static_cast<uint64_t>(row_tile * 4 + wave) * stages * kStageSums + lane % 32 * 4;
  constexpr int kStageGroups = GROUP_WORDS == 4 ? 2 : 1;
  constexpr int kCopies = static_cast<int>(kStageBytes / 1024) + 3 + (LOWS ? 1 : 0);  // of a wave and stage, at least
  const auto fetch = [&](uint32_t stage, bool factors) {
    ManyStage& to_stage = lds[(stage - from) % kManyBuffers];
#pragma unroll
    for (int n = 0; n < static_cast<int>(kStageBytes / 1024); ++n)
      to_lds16(my_x + static_cast<uint64_t>(stage) * kStageBytes + n * 1024, to_stage.x[wave] + n * 1024);
    if (lane < (factors ? 32 : 16)) to_lds16(my_sums + static_cast<uint64_t>(stage) * kStageSums, to_stage.sums[wave]);
    if ((stage + 1) * kStageWords <= p.words) {
      to_lds16(codes + my_codes + stage * kStageWords + lane % 2 * 4, to_stage.codes[wave]);
    } else {
      // x is 0 behind the end of a row; nothing is read behind the last one's
#pragma unroll
      for (int n = 0; n < 4; ++n)
        to_lds4(codes + static_cast<uint64_t>(min(first_out + n * 8 + lane / 8, p.out - 1)) * p.words +
                    min(stage * kStageWords + lane % 8, p.words - 1),
                to_stage.codes[wave][n * 8]);
    }
    const uint32_t group = min(stage * kStageWords / GROUP_WORDS + (kStageGroups == 2 ? lane / 32 : 0), p.groups - 1);
    to_lds4(p.steps + my_groups + group, to_stage.steps[wave]);
    if (LOWS) to_lds4(p.lows + my_groups + group, to_stage.lows[wave]);
  };

  static_assert(kManyRows / kSplitRows * kSplitParts == kWave, "a lane a word");
  const uint32_t some = apart[row_tile * kWave + lane];  // asked for in front of the copies, looked at behind the first of them

  v16f acc[2][2], run[2][2];  // [32 rows][32 outputs]
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[m][n][r] = run[m][n][r] = 0.f;
  // A stage's operands in registers.
  struct Operands {
    v8h hi[2][4], lo[2][4], codes[2][4];
  };
  v16f sum[2][kStageGroups];
  const auto read = [&](uint32_t stage, Operands& k) {
    const ManyStage& here = lds[(stage - from) % kManyBuffers];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const v4u w = here.codes[wave_out * 2 + n][j][half];
      uint32_t a0 = w[0], a1 = w[1], a2 = w[2], a3 = w[3];
      swap32(a0, a2), swap32(a1, a3);  // words (0, 2) (1, 3) (4, 6) (5, 7) of the stage
      k.codes[n][0] = operand_of(a0), k.codes[n][1] = operand_of(a1), k.codes[n][2] = operand_of(a2), k.codes[n][3] = operand_of(a3);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const v8h* at = reinterpret_cast<const v8h*>(here.x[wave_rows * 2 + m]) + t * kWave + lane;
        k.hi[m][t] = at[0], k.lo[m][t] = at[kStageBytes / 32];
      }
  };
  const auto read_sums = [&](uint32_t stage) {
    const ManyStage& here = lds[(stage - from) % kManyBuffers];
#pragma unroll
    for (int u = 0; u < kStageGroups; ++u)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const v4f q = *reinterpret_cast<const v4f*>(&here.sums[wave_rows * 2 + m][u * 32 + 8 * c + 4 * half]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[m][u][4 * c + r] = q[r];
        }
  };
  const auto work = [&](uint32_t stage, const Operands& k, bool opens, bool closes, auto factors) {
    const ManyStage& here = lds[(stage - from) % kManyBuffers];
#pragma unroll
    for (int u = 0; u < kStageGroups; ++u) {
#pragma unroll
      for (int t = u * 4 / kStageGroups; t < (u + 1) * 4 / kStageGroups; ++t)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const v16f zero = {};
            const bool first = opens && t == u * 4 / kStageGroups;
            run[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.hi[m][t], k.codes[n][t],
                                                               first ? (LOWS ? zero : sum[m][u]) : run[m][n], 0, 0, 0);
            run[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.lo[m][t], k.codes[n][t], run[m][n], 0, 0, 0);
          }
      if (closes) {
        if constexpr (factors) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const v16f f = lds_rows(&here.sums[wave_rows * 2 + m][64 + u * 32 + 4 * half]);
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
              for (int n = 0; n < 2; ++n) run[m][n][r] *= f[r];
          }
        }
        const v2f step = lds_pair(&here.steps[wave_out * 2][u * 32 + j]), low = LOWS ? lds_pair(&here.lows[wave_out * 2][u * 32 + j]) : step;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              acc[m][n][r] = __builtin_fmaf(run[m][n][r], step[n], acc[m][n][r]);
              if (LOWS) acc[m][n][r] = __builtin_fmaf(sum[m][u][r], low[n], acc[m][n][r]);
            }
      }
    }
  };
  // two stages are on their way while one is worked on; `from` and `to` are even and differ, a group of 128 is two stages
  constexpr bool kEvery = GROUP_WORDS < 16;  // stage has groups of its own
  const auto all = [&](auto factors) {
    for (uint32_t stage = from; stage < to; stage += 2) {
      copies_done<kCopies>();
      if (stage + 2 < to) fetch(stage + 2, factors);
      Operands k;
      read_sums(stage);
      read(stage, k);
      work(stage, k, true, kEvery, factors);
      if (stage + 2 < to) copies_done<kCopies>();
      else copies_done<0>();
      if (stage + 3 < to) fetch(stage + 3, factors);
      if (kEvery) read_sums(stage + 1);
      read(stage + 1, k);
      work(stage + 1, k, kEvery, true, factors);
    }
  };
  asm volatile("" ::: "memory");
  fetch(from, true), fetch(from + 1, true);
  copies_done<kCopies>();
  // Factors of groups, where any of the 128 rows has one: a loop of its own, since looking for them in every group takes 6 % of
  // 700 rows on 4096 x 4096 weights, 11 % with groups of 64.
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(some != 0) == 0, 1)) all(std::false_type());
  else all(std::true_type());
  // everything is loaded in front of the first store: a load behind one waits for it
  v4f back[2][4];
  float bias[2];
  uint32_t out[2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      back[m][c] = *reinterpret_cast<const v4f*>(undo + row_tile * kManyRows + (wave_rows * 2 + m) * 32 + 8 * c + 4 * half);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    out[n] = out_tile * kManyOut + wave_out * 64 + n * 32 + j;
    bias[n] = p.bias ? p.bias[min(out[n], p.out - 1)] : 0.f;
  }
  loads_done();  // or every store would wait for the one in front of it
  float* const to_y = splits > 1 ? partial + static_cast<uint64_t>(part) * p.rows * p.out : y;
  const bool with_bias = splits == 1 && p.bias;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t row = row_tile * kManyRows + (wave_rows * 2 + m) * 32 + 8 * (r / 4) + 4 * half + r % 4;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float v = acc[m][n][r] * back[m][r / 4][r % 4];
        if (row < p.rows && out[n] < p.out) to_y[static_cast<uint64_t>(row) * p.out + out[n]] = with_bias ? v + bias[n] : v;
      }
    }
}

__global__ __launch_bounds__(kStream) void connected4_join_kernel(const float* partial, float* y, uint32_t count, uint32_t splits,
                                                                  const float* bias, FastDiv f_out) {
  const uint32_t i = blockIdx.x * kStream + threadIdx.x;
  if (i >= count) return;
  float v = partial[i];
  for (uint32_t s = 1; s < splits; ++s) v += partial[static_cast<uint64_t>(s) * count + i];
  if (bias) {
    uint32_t row, o;
    fd_divmod(i, f_out, row, o);
    v += bias[o];
  }
  y[i] = v;
}

struct ManyPlan {
  uint32_t row_tiles, out_tiles, stages, splits;
  size_t parts_bytes, sums_bytes, undo_bytes, apart_bytes, partial_bytes;
  size_t bytes() const { return parts_bytes + sums_bytes + undo_bytes + apart_bytes + partial_bytes; }
};
// Which kernel, by what it costs: 16 rows at a time 4 us and 0.165 for a million weights and set of 16, tiles 15 us (two or three launches, few
// of them whole on the chip) and 0.8 for a million weights and 128 rows.  4096 x 4096 weights: 128 rows 23.3 us by 16 and 29.0 in
// tiles, 256 rows 43.2 and 38.5; 16384 x 4096: 64 rows 54.0 and 61.9, 96 rows 76.8 and 64.4; 1024 x 1024: 256 rows 8.8 and 18.7.  Grids have up to
// 65535 rows.
static bool many(int rows, int in, int out) {
  if (rows <= 64) return false;  // the difference below is not positive
  const int64_t sets = (rows + 15) / 16, tiles = (rows + 127) / 128;
  return rows > 4096 || static_cast<int64_t>(in) * out * (165 * sets - 800 * tiles) > int64_t{11000} << 20;
}
static ManyPlan plan_many(int rows, int in, int out) {
  ManyPlan m;
  m.row_tiles = (static_cast<uint32_t>(rows) + kManyRows - 1) / kManyRows;
  m.out_tiles = (static_cast<uint32_t>(out) + kManyOut - 1) / kManyOut;
  m.stages = ((static_cast<uint32_t>(in) / 8 + kStageWords - 1) / kStageWords + 1) & ~1u;  // whole groups of 128
  // parts of `in`, where tiles alone do not fill the chip: none under 512 codes
  const uint64_t tiles = static_cast<uint64_t>(m.row_tiles) * m.out_tiles;
  m.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(256 / tiles, m.stages / 8)));
  m.parts_bytes = static_cast<size_t>(m.row_tiles) * 4 * m.stages * kStageBytes;
  m.sums_bytes = static_cast<size_t>(m.row_tiles) * 4 * m.stages * kStageSums * sizeof(float);
  m.undo_bytes = static_cast<size_t>(m.row_tiles) * kManyRows * sizeof(float);
  m.apart_bytes = static_cast<size_t>(m.row_tiles) * kWave * sizeof(uint32_t);
  m.partial_bytes = m.splits == 1 ? 0 : static_cast<size_t>(m.splits) * rows * out * sizeof(float);
  return m;
}

template <int GROUP_WORDS, bool LOWS>
static int launch_many(const ManyPlan& m, const float* x, const uint32_t* codes, float* y, void* workspace, const Connected4Args& p,
                       hipStream_t st) {
  char* at = static_cast<char*>(workspace);
  v8h* parts = reinterpret_cast<v8h*>(at);
  float* sums = reinterpret_cast<float*>(at + m.parts_bytes);
  float* undo = reinterpret_cast<float*>(at + m.parts_bytes + m.sums_bytes);
  uint32_t* apart = reinterpret_cast<uint32_t*>(at + m.parts_bytes + m.sums_bytes + m.undo_bytes);
  float* partial = reinterpret_cast<float*>(at + m.parts_bytes + m.sums_bytes + m.undo_bytes + m.apart_bytes);
  const dim3 split_grid(m.row_tiles * kManyRows / kSplitRows, kSplitParts);
  connected4_split_kernel<GROUP_WORDS, LOWS><<<split_grid, kBlock, 0, st>>>(x, parts, sums, undo, apart, p.rows, p.words, m.stages);
  if (int rc = launch_status()) return rc;
  connected4_many_kernel<GROUP_WORDS, LOWS><<<m.row_tiles * m.out_tiles * m.splits, kBlock, 0, st>>>(
      parts, sums, undo, apart, codes, y, partial, m.stages, m.splits, m.row_tiles, p);
  if (int rc = launch_status()) return rc;
  if (m.splits > 1) {
    const uint32_t count = p.rows * p.out;
    connected4_join_kernel<<<stream_grid(count), kStream, 0, st>>>(partial, y, count, m.splits, p.bias, make_fastdiv(p.out));
  }
  return launch_status();
}

struct FewPlan {
  bool own, digits;
  uint32_t sets, blocks;
  size_t set_parts, set_factors;  // bytes, floats
  size_t bytes() const { return own ? 0 : sets * (set_parts + set_factors * sizeof(float)); }
};
static FewPlan plan_few(int rows, int in, int group) {
  FewPlan f;
  // 6144 outputs of 4096 for one row 6.3 us, 8.4 with the digits from a launch of their own; 32000 of 4096 17.2 and 22.1.  Of four
  // rows they cost each workgroup more than that launch (4096 outputs of 4096 8.5 us, 7.0 with the launch).
  f.own = rows == 1;
  f.digits = rows <= 8;  // 8 rows on 16384 x 4096 weights 18.1 us with digits, 24.1 with halves; 6 on 4096 x 4096 7.9 and 8.8
  f.sets = f.digits ? 1 : (static_cast<uint32_t>(rows) + 15) / 16;
  f.blocks = (static_cast<uint32_t>(in) / 8 + kBlockWords - 1) / kBlockWords;
  const size_t groups = static_cast<size_t>(f.blocks) * (kBlockWords * 8 / group);
  const size_t fours = f.digits ? (rows + 3) / 4 : 4;
  f.set_parts = f.blocks * (f.digits ? fours * kFewBlockBytes : 4 * 4 * 16 * 32);
  f.set_factors = groups * 8 * fours;
  return f;
}

template <class ROWS, int GROUP_WORDS, int TILES, bool LOWS>
static int launch_few_of(const float* x, const char* parts, const float* factors, const uint32_t* codes, float* y, const FewPlan& f,
                         const Connected4Args& p, hipStream_t st) {
  const dim3 grid((p.out + 16 * TILES - 1) / (16 * TILES), f.sets);
  constexpr uint32_t kEach = ROWS::kGroups * (16 * TILES * (LOWS ? 2 : 1) + ROWS::kFactors) + ROWS::kFloats;  // floats of a block
  const uint32_t chunks = (f.blocks + kFewFloats / kEach - 1) / (kFewFloats / kEach), chunk = (f.blocks + chunks - 1) / chunks;
  const uint32_t bytes = std::max<uint32_t>(chunk * kEach + 32 * TILES, kFewWaves * TILES * ROWS::kSums * kWave) * sizeof(float);
  connected4_few_kernel<ROWS, GROUP_WORDS, TILES, LOWS>
      <<<grid, kFewWaves * kWave, bytes, st>>>(x, parts, factors, codes, y, f.blocks, chunk, f.set_parts, f.set_factors, p);
  return launch_status();
}
template <int GROUP_WORDS, bool LOWS>
static int launch_few(const float* x, const uint32_t* codes, float* y, void* workspace, const Connected4Args& p, hipStream_t st) {
  const FewPlan f = plan_few(p.rows, p.words * 8, GROUP_WORDS * 8);
  // One row: one tile of outputs a workgroup (32000 outputs 17.0 us, 18.1 with two, 8192 7.0 and 7.2).  Up to 8 rows: one, or two where
  // that still fills the chip twice: 16384 outputs for four rows 16.6 us with two and 17.9 with one, for eight 16.6 and 20.0; 8192
  // for four 10.4 and 9.8, for eight 11.4 and 11.5.  More rows: as many of one, two and four as leave a workgroup for
  // each compute unit, since each reads all of x: 16384 outputs for 16 rows 19.5 us with four, 23 with two, 26.5 with one; 4096 for 32 rows
  // 13.2, 10.1 and 11.9.
  const auto wide = [&](uint32_t outputs) { return (p.out + outputs - 1) / outputs * f.sets >= 256; };
  const bool two = p.out >= 16 * 512;
  if (f.own) return launch_few_of<OneRow<GROUP_WORDS, LOWS>, GROUP_WORDS, 1, LOWS>(x, nullptr, nullptr, codes, y, f, p, st);
  char* parts = static_cast<char*>(workspace);
  float* factors = reinterpret_cast<float*>(parts + f.sets * f.set_parts);
  const dim3 grid((f.blocks * kBlockWords + kBlock - 1) / kBlock, p.rows);
  if (f.digits)
    connected4_digits_kernel<GROUP_WORDS, LOWS><<<grid, kBlock, 0, st>>>(x, parts, factors, p.words, f.blocks, (p.rows + 3) / 4);
  else
    connected4_halves_kernel<GROUP_WORDS, LOWS><<<grid, kBlock, 0, st>>>(x, parts, factors, p.words, f.blocks);
  if (int rc = launch_status()) return rc;
  if (!f.digits) {
    if (wide(64)) return launch_few_of<HalfRows<GROUP_WORDS, LOWS>, GROUP_WORDS, 4, LOWS>(x, parts, factors, codes, y, f, p, st);
    if (wide(32)) return launch_few_of<HalfRows<GROUP_WORDS, LOWS>, GROUP_WORDS, 2, LOWS>(x, parts, factors, codes, y, f, p, st);
    return launch_few_of<HalfRows<GROUP_WORDS, LOWS>, GROUP_WORDS, 1, LOWS>(x, parts, factors, codes, y, f, p, st);
  }
  if (p.rows <= 4)
    return two ? launch_few_of<DigitRows<GROUP_WORDS, 1, LOWS>, GROUP_WORDS, 2, LOWS>(x, parts, factors, codes, y, f, p, st)
               : launch_few_of<DigitRows<GROUP_WORDS, 1, LOWS>, GROUP_WORDS, 1, LOWS>(x, parts, factors, codes, y, f, p, st);
  return two ? launch_few_of<DigitRows<GROUP_WORDS, 2, LOWS>, GROUP_WORDS, 2, LOWS>(x, parts, factors, codes, y, f, p, st)
             : launch_few_of<DigitRows<GROUP_WORDS, 2, LOWS>, GROUP_WORDS, 1, LOWS>(x, parts, factors, codes, y, f, p, st);
}

static bool connected4_shape(int rows, int in, int out) {
  return rows >= 0 && out >= 0 && in >= 8 && in % 8 == 0 && static_cast<int64_t>(rows) * out <= INT32_MAX &&
         static_cast<int64_t>(rows) * in <= INT32_MAX;
}
// Offsets within a workgroup's up to 64 outputs have 32 bits (64 outputs of 2^26 words are 2^32), and so have the lanes of a grid.
static bool connected4_extents(int rows, int in, int out) { return rows <= 1 << 26 && in <= 1 << 29 && out <= 1 << 26; }
static bool connected4_group(int group) { return group == 32 || group == 64 || group == 128; }

}  // namespace shdw

using namespace shdw;

extern "C" {

size_t shdw_hip_connected4_workspace_bytes(int rows, int in, int out, int group) {
  if (!connected4_shape(rows, in, out) || !connected4_group(group) || !connected4_extents(rows, in, out) || rows == 0 || out == 0)
    return 0;
  return many(rows, in, out) ? plan_many(rows, in, out).bytes() : plan_few(rows, in, group).bytes();
}

int shdw_hip_connected4(int rows, int in, int out, int group, const float* x, const int* codes, const float* steps,
                        const float* lows, const float* bias, float* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (!connected4_shape(rows, in, out)) return SHDW_E_INVALID_ARGUMENT;
  if (!connected4_group(group) || !connected4_extents(rows, in, out)) return SHDW_E_UNSUPPORTED;
  if (rows == 0 || out == 0) return SHDW_OK;
  if (!x || !codes || !steps || !y || x == y) return SHDW_E_INVALID_ARGUMENT;
  Connected4Args p;
  p.rows = static_cast<uint32_t>(rows), p.words = static_cast<uint32_t>(in / 8), p.out = static_cast<uint32_t>(out);
  p.groups = static_cast<uint32_t>((in + group - 1) / group);
  p.steps = steps, p.lows = lows, p.bias = bias;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(codes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (const size_t need = shdw_hip_connected4_workspace_bytes(rows, in, out, group)) {
    if (!workspace || workspace_bytes < need) return SHDW_E_WORKSPACE;
    if (!aligned16(workspace)) return SHDW_E_INVALID_ARGUMENT;
  }
  if (many(rows, in, out)) {
    const ManyPlan m = plan_many(rows, in, out);
    if (group == 32)
      return lows ? launch_many<4, true>(m, x, words, y, workspace, p, st) : launch_many<4, false>(m, x, words, y, workspace, p, st);
    if (group == 64)
      return lows ? launch_many<8, true>(m, x, words, y, workspace, p, st) : launch_many<8, false>(m, x, words, y, workspace, p, st);
    return lows ? launch_many<16, true>(m, x, words, y, workspace, p, st) : launch_many<16, false>(m, x, words, y, workspace, p, st);
  }
  if (group == 32) return lows ? launch_few<4, true>(x, words, y, workspace, p, st) : launch_few<4, false>(x, words, y, workspace, p, st);
  if (group == 64) return lows ? launch_few<8, true>(x, words, y, workspace, p, st) : launch_few<8, false>(x, words, y, workspace, p, st);
  return lows ? launch_few<16, true>(x, words, y, workspace, p, st) : launch_few<16, false>(x, words, y, workspace, p, st);
}

}  // extern "C"
