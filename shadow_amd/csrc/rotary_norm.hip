// RotaryNorm: the packed projections of a layer's queries, keys and values,
// x [batch][length][q_heads + 2 * kv_heads][head_dim], taken apart.  Every head of a query or a
// key is divided by its root mean square and multiplied by a learned scale,
//   y[d] = x[d] / sqrt(mean(x^2) + eps) * scale[d],
// then pairs of it are turned by an angle that grows with the token's position,
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * frequency[pair];
// values are copied.  Queries go to a tensor of their own, keys and values to the rows of two
// caches (or to dense tensors).  The reference has no such operator.
//
// The angle reaches 10^6 and more while cos and sin look at what is left of it after whole turns:
// the product and the turns are formed in fp64 (a position has 31 bits, a frequency 24), the rest,
// at most half a turn, goes to fp32 sincospi.
//
// Bound by its bytes: two prompts of up to 4096 tokens, 48 heads of 128 values, 63 us, 5.1 TB/s (a large copy: 4.8); one token 3.7 us, a launch.
// That is heads of up to 256 values and a rotated part that are whole vectors (rotary_heads_kernel).  Any other head takes
// rotary_norm_kernel, a wave a head, which works the angles out for each and goes through LDS: the same prompts with heads of 126
// values 282 us, of 128 with 36 of them turned 243, of 512 915.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/shadow_hip.h"
#include "device_common.h"
#include "launch.h"

#pragma clang fp contract(off)

namespace shdw {

constexpr int kRotaryMaxDim = 1024;

struct RotaryArgs {
  int length, q_heads, kv_heads, dim, rotary, interleaved, normalize, capacity;
  float eps, inv_dim;
  const float* q_scale;
  const float* k_scale;
  const float* frequency;
  const int* starts;
  const int* lengths;
  FastDiv f_heads, f_length;
};

// cos and sin of position * frequency.
SHDW_DEVICE void turn(int64_t position, float frequency, float& c, float& s) {
  const double turns = static_cast<double>(position) * static_cast<double>(frequency) * 0.15915494309189533577;
  const float rest = static_cast<float>(turns - __builtin_rint(turns));
  sincospif(rest + rest, &s, &c);
}

// Whether a mean of squares (and eps) in fp32 is one that nothing was lost in: squares of less than 2^-126 are, and so is a sum
// of more than fp32 holds.  Heads of such sizes, or of zeros with an eps as small, take their mean in fp64.
SHDW_DEVICE bool exact_mean(float mean) { return mean >= 0x1p-90f && mean < INFINITY; }
SHDW_DEVICE double norm_factor(double sum, int dim, float eps) { return 1.0 / __builtin_sqrt(sum / dim + static_cast<double>(eps)); }

// Where head h of token (b, t) goes; nullptr where nothing is written.
SHDW_DEVICE float* rotary_target(const RotaryArgs& p, float* q, float* k, float* v, uint32_t b, uint32_t t, uint32_t h,
                                 int64_t position) {
  const uint32_t q_heads = static_cast<uint32_t>(p.q_heads), kv = static_cast<uint32_t>(p.kv_heads);
  if (h < q_heads) return q + ((static_cast<uint64_t>(b) * p.length + t) * q_heads + h) * p.dim;
  const bool is_v = h >= q_heads + kv;
  const uint32_t kh = h - q_heads - (is_v ? kv : 0u);
  const int64_t row = p.capacity > 0 ? position : t, rows = p.capacity > 0 ? p.capacity : p.length;
  if (row < 0 || row >= rows) return nullptr;
  return (is_v ? v : k) + ((static_cast<uint64_t>(b) * kv + kh) * rows + row) * p.dim;
}

// Heads whose values and halves are whole vectors: LANES lanes a head, four values a lane, so a wave takes
// 64 / LANES heads at a time; it takes one token and one of `parts` parts of its heads, four turns' loads
// under way at once.  The angles are worked out once for all of them.  MODE 0: no rotation, 1: halves, 2: neighbours.
template <int LANES>
SHDW_DEVICE float across_head(float v) {
  v += dpp_f32<kDppXor1>(v);
  v += dpp_f32<kDppXor2>(v);
  v += dpp_f32<kDppHalfMirror>(v);
  v += dpp_f32<kDppMirror>(v);
  if (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (LANES >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Four values of a head over its norm in fp64.  Rare and long, so out of line: in line two prompts take 63.5 us for 62.8.
template <int LANES>
__device__ __attribute__((noinline)) v4f wide_norm(v4f e, int dim, float eps) {
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < 4; ++c) sum += static_cast<double>(e[c]) * e[c];
  for (int step = 1; step < LANES; step <<= 1) sum += __shfl_xor(sum, step);
  const double f = norm_factor(sum, dim, eps);
  return v4f{static_cast<float>(e[0] * f), static_cast<float>(e[1] * f), static_cast<float>(e[2] * f), static_cast<float>(e[3] * f)};
}

template <int LANES, int MODE>
__global__ __launch_bounds__(kBlock) void rotary_heads_kernel(const float* x, float* q, float* k, float* v, uint32_t parts,
                                                              uint32_t waves, RotaryArgs p) {
  constexpr int kHeads = kWave / LANES, kTurns = 4;
  const uint32_t lane = threadIdx.x % kWave, u = lane % LANES, sub = lane / LANES;
  const uint32_t item = blockIdx.x * (kBlock / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (item >= waves) return;
  const uint32_t token = item / parts, part = item % parts;
  uint32_t b, t;
  fd_divmod(token, p.f_length, b, t);
  const int count = p.lengths ? p.lengths[b] : p.length;
  if (static_cast<int>(t) >= count) return;
  const int64_t position = static_cast<int64_t>(p.starts ? p.starts[b] : 0) + t;
  const int64_t row = p.capacity > 0 ? position : t, rows = p.capacity > 0 ? p.capacity : p.length;
  const bool kept = row >= 0 && row < rows;  // by the caches

  const int d = 4 * u, half = p.rotary / 2;
  const bool there = d < p.dim, turned = MODE != 0 && d < p.rotary;
  // what a lane's values are turned by, and with which lane's
  float cosine[4] = {1.f, 1.f, 1.f, 1.f}, sine[4] = {};
  const bool second = MODE == 1 && d >= half;
  const int other = MODE == 1 ? (sub * LANES + u + (second ? -half : half) / 4) & (kWave - 1) : 0;
  if (turned) {
    if (MODE == 1) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        turn(position, p.frequency[(second ? d - half : d) + c], cosine[c], sine[c]);
        if (!second) sine[c] = -sine[c];
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        turn(position, p.frequency[(d + c) / 2], cosine[c], sine[c]);
        cosine[c + 1] = cosine[c], sine[c + 1] = sine[c], sine[c] = -sine[c];
      }
    }
  }
  v4f q_scale = {1.f, 1.f, 1.f, 1.f}, k_scale = q_scale;
  if (p.normalize && there) {
    if (p.q_scale) q_scale = load4_any(p.q_scale + d);
    if (p.k_scale) k_scale = load4_any(p.k_scale + d);
  }

  const uint32_t q_heads = p.q_heads, kv = p.kv_heads, heads = q_heads + 2 * kv;
  const uint32_t turns = (heads + kHeads - 1) / kHeads;
  const uint32_t from = turns * part / parts, to = turns * (part + 1) / parts;
  const float* in = x + static_cast<uint64_t>(token) * heads * p.dim + d;
  float* q_out = q + static_cast<uint64_t>(token) * q_heads * p.dim + d;
  const uint64_t head_size = static_cast<uint64_t>(rows) * p.dim;
  const uint64_t cache = (static_cast<uint64_t>(b) * kv * rows + static_cast<uint64_t>(row)) * p.dim + d;
  for (uint32_t turn0 = from; turn0 < to; turn0 += kTurns) {
    v4f e[kTurns];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      const uint32_t h = (turn0 + n) * kHeads + sub;
      e[n] = turn0 + n < to && h < heads && there ? load4_stream_any(in + static_cast<uint64_t>(h) * p.dim) : v4f{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      if (turn0 + n >= to) break;
      const uint32_t h = (turn0 + n) * kHeads + sub;
      const bool is_q = h < q_heads, is_v = h >= q_heads + kv;
      v4f y = e[n];
      if (p.normalize) {
        float sum = e[n][0] * e[n][0];
#pragma unroll
        for (int c = 1; c < 4; ++c) sum = __builtin_fmaf(e[n][c], e[n][c], sum);
        sum = across_head<LANES>(sum);
        const float mean = __builtin_fmaf(sum, p.inv_dim, p.eps), f = 1.f / __builtin_sqrtf(mean);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = e[n][c] * f;
        const bool off = !exact_mean(mean) && h < heads && !is_v;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(off) != 0, 0)) {
          const v4f wide = wide_norm<LANES>(e[n], p.dim, p.eps);
          if (off) y = wide;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] *= is_q ? q_scale[c] : k_scale[c];
      }
      if (MODE != 0) {
        v4f o;
        if (MODE == 1) {
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] = __shfl(y[c], other);
        } else {
          o = v4f{y[1], y[0], y[3], y[2]};
        }
        if (turned) {
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] = __builtin_fmaf(y[c], cosine[c], o[c] * sine[c]);
        }
      }
      if (is_v) y = e[n];
      if (h < heads && there && (is_q || kept)) {
        float* out = is_q ? q_out + static_cast<uint64_t>(h) * p.dim
                          : (is_v ? v : k) + cache + (h - q_heads - (is_v ? kv : 0u)) * head_size;
        store4_stream_any(out, y);
      }
    }
  }
}

// A wave a head, any head_dim of up to 1024.
__global__ __launch_bounds__(kBlock) void rotary_norm_kernel(const float* x, float* q, float* k, float* v, uint32_t items,
                                                             RotaryArgs p) {
  extern __shared__ float lds[];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t item = blockIdx.x * (kBlock / kWave) + wave;
  if (item >= items) return;  // no barrier below: a wave works on its own part of the LDS
  uint32_t token, h, b, t;
  fd_divmod(item, p.f_heads, token, h);
  fd_divmod(token, p.f_length, b, t);
  const int count = p.lengths ? p.lengths[b] : p.length;
  if (static_cast<int>(t) >= count) return;
  const int64_t position = static_cast<int64_t>(p.starts ? p.starts[b] : 0) + t;
  float* out = rotary_target(p, q, k, v, b, t, h, position);
  if (out == nullptr) return;
  const float* in = x + static_cast<uint64_t>(item) * p.dim;
  const int dim = p.dim;
  if (h >= static_cast<uint32_t>(p.q_heads + p.kv_heads)) {
    for (int d = lane; d < dim; d += kWave) out[d] = in[d];
    return;
  }
  float* head = lds + wave * dim;
  float sum = 0.f;
  for (int d = lane; d < dim; d += kWave) {
    const float e = in[d];
    head[d] = e;
    sum = __builtin_fmaf(e, e, sum);
  }
  for (int step = 1; step < kWave; step <<= 1) sum += __shfl_xor(sum, step);
  float factor = 1.f;
  if (p.normalize) {
    const float mean = __builtin_fmaf(sum, p.inv_dim, p.eps);
    if (exact_mean(mean)) {
      factor = 1.f / __builtin_sqrtf(mean);
    } else {
      double wide = 0.0;
      for (int d = lane; d < dim; d += kWave) wide += static_cast<double>(head[d]) * head[d];
      for (int step = 1; step < kWave; step <<= 1) wide += __shfl_xor(wide, step);
      const double f = norm_factor(wide, p.dim, p.eps);
      for (int d = lane; d < dim; d += kWave) head[d] = static_cast<float>(head[d] * f);
    }
  }
  const float* scale = !p.normalize ? nullptr : h < static_cast<uint32_t>(p.q_heads) ? p.q_scale : p.k_scale;
  const int half = p.rotary / 2;
  const auto value = [&](int d) { return scale ? head[d] * factor * scale[d] : head[d] * factor; };
  for (int d = lane; d < dim; d += kWave) {
    float y = value(d);
    if (d < p.rotary) {
      const int pair = p.interleaved ? d >> 1 : d < half ? d : d - half;
      const bool second = p.interleaved ? d & 1 : d >= half;
      const float other = value(p.interleaved ? d ^ 1 : second ? d - half : d + half);
      float c, s;
      turn(position, p.frequency[pair], c, s);
      y = second ? __builtin_fmaf(y, c, other * s) : __builtin_fmaf(y, c, -(other * s));
    }
    out[d] = y;
  }
}

}  // namespace shdw

using namespace shdw;

extern "C" {

int shdw_hip_rotary_norm(int batch, int length, int q_heads, int kv_heads, int head_dim, int rotary_dim, int interleaved,
                         int normalize, float eps, const float* x, const float* q_scale, const float* k_scale,
                         const float* frequency, const int* starts, const int* lengths, int capacity, float* q, float* k,
                         float* v, void* stream) {
  if (batch < 0 || length < 0 || q_heads < 0 || kv_heads < 0 || head_dim < 1 || capacity < 0) return SHDW_E_INVALID_ARGUMENT;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0) return SHDW_E_INVALID_ARGUMENT;
  if (normalize && !(eps >= 0.f)) return SHDW_E_INVALID_ARGUMENT;
  if (head_dim > kRotaryMaxDim) return SHDW_E_UNSUPPORTED;
  const int64_t heads = static_cast<int64_t>(q_heads) + 2 * static_cast<int64_t>(kv_heads);
  if (batch == 0 || length == 0 || heads == 0) return SHDW_OK;
  const int64_t tokens = static_cast<int64_t>(batch) * length;
  // indexes of heads and products of two counts of turns have 32 bits
  if (tokens > INT32_MAX || heads > 1 << 18 || tokens * heads > INT32_MAX) return SHDW_E_UNSUPPORTED;
  if (!x || (q_heads > 0 && !q) || (kv_heads > 0 && (!k || !v)) || (rotary_dim > 0 && !frequency)) return SHDW_E_INVALID_ARGUMENT;
  if (x == q || x == k || x == v || (kv_heads > 0 && (k == v || (q_heads > 0 && (q == k || q == v)))))
    return SHDW_E_INVALID_ARGUMENT;
  RotaryArgs p;
  p.length = length, p.q_heads = q_heads, p.kv_heads = kv_heads, p.dim = head_dim, p.rotary = rotary_dim;
  p.interleaved = interleaved != 0, p.normalize = normalize != 0, p.capacity = capacity;
  p.eps = eps, p.inv_dim = 1.f / head_dim;
  p.q_scale = q_scale, p.k_scale = k_scale, p.frequency = frequency, p.starts = starts, p.lengths = lengths;
  p.f_heads = make_fastdiv(static_cast<uint32_t>(heads)), p.f_length = make_fastdiv(static_cast<uint32_t>(length));
  constexpr uint32_t kWaves = kBlock / kWave;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (head_dim <= 256 && head_dim % 4 == 0 && rotary_dim % (interleaved ? 4 : 8) == 0) {
    const int lanes = head_dim <= 64 ? 16 : head_dim <= 128 ? 32 : 64;
    // parts of a token's heads: enough waves to fill the chip, a turn each at least
    const int64_t turns = (heads * lanes + kWave - 1) / kWave;
    const uint32_t parts = static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(turns, 8192 / tokens)));
    const uint32_t waves = static_cast<uint32_t>(tokens) * parts;
    if (!grid_fits((waves + kWaves - 1) / kWaves, kBlock)) return SHDW_E_UNSUPPORTED;
    const int mode = rotary_dim == 0 ? 0 : interleaved ? 2 : 1;
    void (*kernel)(const float*, float*, float*, float*, uint32_t, uint32_t, RotaryArgs) =
        lanes == 16   ? (mode == 0 ? rotary_heads_kernel<16, 0> : mode == 1 ? rotary_heads_kernel<16, 1> : rotary_heads_kernel<16, 2>)
        : lanes == 32 ? (mode == 0 ? rotary_heads_kernel<32, 0> : mode == 1 ? rotary_heads_kernel<32, 1> : rotary_heads_kernel<32, 2>)
                      : (mode == 0 ? rotary_heads_kernel<64, 0> : mode == 1 ? rotary_heads_kernel<64, 1> : rotary_heads_kernel<64, 2>);
    kernel<<<(waves + kWaves - 1) / kWaves, kBlock, 0, st>>>(x, q, k, v, parts, waves, p);
    return launch_status();
  }
  const uint32_t items = static_cast<uint32_t>(tokens * heads);
  if (!grid_fits((items + kWaves - 1) / kWaves, kBlock)) return SHDW_E_UNSUPPORTED;
  rotary_norm_kernel<<<(items + kWaves - 1) / kWaves, kBlock, kWaves * head_dim * sizeof(float), st>>>(x, q, k, v, items, p);
  return launch_status();
}

}  // extern "C"
