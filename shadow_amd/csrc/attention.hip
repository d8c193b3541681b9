// WindowAttention: y = softmax(scale * q k^T over the visible keys) v for every query of
// q [batch][length][q_heads][head_dim] on caches k, v [batch][kv_heads][capacity][head_dim];
// q_heads / kv_heads heads share a key head.  Query t of sequence b stands at position
// starts[b] + t, the caches hold min(starts[b] + lengths[b], capacity) rows of it.  Visible is
// what lies within the window (0: no limit) and, under `causal`, not behind the query; the first
// `sinks` keys stay visible outside the window.  A query that sees nothing gives zeros.  The
// reference has no such operator.
//
// The rows of a key head are its queries and the heads that share it, row = t * group + head.
// One pass over the keys carries a running maximum and sum; scores are held in powers of two,
// log2(e) being part of the scale.
//
// Few rows (a token, or a few): the caches are read once and that is the time.  A wave takes
// tiles of 16 keys for 16 rows on the fp32 matrix instruction 16x16x4, operands straight from
// memory: lane l = 16 g + i reads values 16 s + 4 g .. + 3 of key i, the four of them are operands
// of four products over dims {16 s + 4 g + c}, in which the rows' values stand the same way.
// Products come out as scores of keys 4 g + r for row i, which is what the weights' operand
// of the second product is, with keys {4 g + r} for its contraction: nothing is moved
// between lanes, nothing goes through LDS before the end.  32 sequences with a token each over up to 4000 keys of 8 heads of 128
// values 132 us (5.4 TB/s of keys and values), one sequence over 65536 keys 85 (6.3 TB/s), over 8192 22, over a window of
// 1024 12.8: two launches, positions that have to be there before keys can be asked for, one tile a wave.
#include "attention_common.h"

#include "../../include/shadow_hip.h"
#include "attention_tiles.h"
#include "launch.h"

#pragma clang fp contract(off)

namespace shdw {

constexpr int kRowsBits = 4;
constexpr int kRowsBlock = 1 << kRowsBits;  // rows of a workgroup of the kernel for few rows
constexpr int kRowsTile = 16;      // keys of its tiles
constexpr int kRowsWaves = 4;      // waves that share its tiles

// Vectors of four values of a row, d in steps of four.  The last one of a row whose length is no multiple of four, and all behind it, is
// the row's last four values: those that another vector has too meet zeros of q and are not stored.  Heads of fewer than
// four values (VECTORS false) are taken value by value.
template <bool VECTORS>
SHDW_DEVICE int first_of(int d, int dim) { return VECTORS ? min(d, dim - 4) : d; }
template <bool VECTORS>
SHDW_DEVICE bool counts(int d, int c, int dim) {
  const int at = first_of<VECTORS>(d, dim) + c;
  return at >= d && at < dim;
}
template <bool VECTORS>
SHDW_DEVICE v4f row4(const float* row, int d, int dim) {
  if (VECTORS) return load4_stream_any(row + first_of<true>(d, dim));
  v4f v;
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = row[min(d + c, dim - 1)];
  return v;
}
template <bool VECTORS>
SHDW_DEVICE void put4(float* row, int d, int dim, v4f v) {
  if (VECTORS && d + 4 <= dim) {
    *reinterpret_cast<v4f_unaligned*>(row + d) = v;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (counts<VECTORS>(d, c, dim)) row[first_of<VECTORS>(d, dim) + c] = v[c];
  }
}

// One tile's keys and values as a lane holds them.
template <int NB>
struct RowsTile {
  v4f k[4 * NB], v[4][NB];
};
template <int NB, bool VECTORS>
SHDW_DEVICE void load_keys(RowsTile<NB>& t, const float* k, int dim, int j0, int end, int g, int i) {
  const float* kr = k + static_cast<uint64_t>(min(j0 + i, end - 1)) * dim;
#pragma unroll
  for (int s = 0; s < 4 * NB; ++s) t.k[s] = row4<VECTORS>(kr, 16 * s + 4 * g, dim);
}
template <int NB, bool VECTORS>
SHDW_DEVICE void load_values(RowsTile<NB>& t, const float* v, int dim, int j0, int end, int g, int i) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float* vr = v + static_cast<uint64_t>(min(j0 + 4 * g + r, end - 1)) * dim;
#pragma unroll
    for (int n = 0; n < NB; ++n) t.v[r][n] = row4<VECTORS>(vr, 64 * n + 4 * i, dim);
  }
}

// A workgroup takes `kRowsBlock` rows of a key head and one of `splits` parts of their tiles; its waves
// take every fourth tile of the part.  With one part it writes y, with more its sums, joined by
// attention_join_kernel: sums of a row over the weights 2^(score - top) and the weighted values.
template <int NB, bool VECTORS>
__global__ __launch_bounds__(kRowsWaves * kWave, NB <= 2 ? 2 : 1) void attention_rows_kernel(
    const float* q, const float* k, const float* v, float* y, float* sums, FastDiv f_splits, FastDiv f_blocks, AttentionArgs p) {
  __shared__ v4f share[2 * 4 * NB * kWave];
  __shared__ float tops[kRowsWaves][kRowsBlock], totals[kRowsWaves][kRowsBlock];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, g = lane / 16, i = lane % 16;
  const uint32_t blocks = f_blocks.d, splits = f_splits.d;
  uint32_t rest, block, head, part, b, h;
  fd_divmod(blockIdx.x, f_blocks, rest, block);
  fd_divmod(rest, f_splits, head, part);
  fd_divmod(head, p.f_kv, b, h);
  const Sequence seq = sequence_of(p, b);
  const int row = block * kRowsBlock + i;                       // this lane's
  const int rows = seq.count * p.group;                         // of the key head
  if (static_cast<int>(block * kRowsBlock) >= rows) return;
  uint32_t t, shared;
  fd_divmod(min(row, rows - 1), p.f_group, t, shared);
  const int t_first = fd_div(block * kRowsBlock, p.f_group), t_last = fd_div(min(rows - 1, static_cast<int>(block * kRowsBlock) + 15), p.f_group);
  const Reach reach = reach_of(p, seq, t);
  const TileList list = tiles_of<kRowsTile>(reach_of(p, seq, t_first), reach_of(p, seq, t_last));
  const bool mine = row < rows;
  const uint64_t at = ((static_cast<uint64_t>(b) * p.length + t) * p.q_heads + h * p.group + shared) * p.dim;

  const float* kh = k + static_cast<uint64_t>(head) * p.capacity * p.dim;
  const float* vh = v + static_cast<uint64_t>(head) * p.capacity * p.dim;

  v4f acc[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[n][c] = v4f{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, total = 0.f;

  int from, to;
  part_of(list.tiles, part, f_splits, from, to);
  // the first tile is on its way before anything is waited for
  // The next tile's keys and values are on their way while one is worked on; of more than 192 dimensions its keys, with the tile's own
  // values (all of them do not fit the registers: 8 tokens over 4000 keys of 4 heads of 256 77 us, 109 with both).
  constexpr bool kBoth = NB < 4;
  RowsTile<NB> now, next;
  int tile = from + wave, j0 = 0, end = 0, j1 = 0, end1 = 0;
  if (tile < to) {
    tile_keys<kRowsTile>(list, tile, j0, end);
    load_keys<NB, VECTORS>(now, kh, p.dim, j0, end, g, i);
    if (kBoth) load_values<NB, VECTORS>(now, vh, p.dim, j0, end, g, i);
  }
  asm volatile("" ::: "memory");
  v4f qv[4 * NB];
#pragma unroll
  for (int s = 0; s < 4 * NB; ++s) {
    const int d = 16 * s + 4 * g;
    const v4f w = row4<VECTORS>(q + at, d, p.dim);
#pragma unroll
    for (int c = 0; c < 4; ++c) qv[s][c] = counts<VECTORS>(d, c, p.dim) ? w[c] * (p.scale * kLog2e) : 0.f;
  }
#pragma unroll 1
  while (tile < to) {
    // loads are made in any case, behind the end one row's: a load that may not be made would have to be waited for as
    // if it were the last
    const bool more = tile + kRowsWaves < to;
    tile_keys<kRowsTile>(list, min(tile + kRowsWaves, to - 1), j1, end1);
    if (!kBoth) load_values<NB, VECTORS>(now, vh, p.dim, j0, end, g, i);
    load_keys<NB, VECTORS>(next, kh, p.dim, j1, more ? end1 : j1 + 1, g, i);
    if (kBoth) load_values<NB, VECTORS>(next, vh, p.dim, j1, more ? end1 : j1 + 1, g, i);
    asm volatile("" ::: "memory");
    v4f s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4 * NB; ++s)
      if (16 * s < p.dim) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(now.k[s][c], qv[s][c], s4, 0, 0, 0);
      }
    const bool whole = all_see<kRowsTile>(list, j0, end);
    if (!whole) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = j0 + 4 * g + r;
        const bool seen = j < end && sees(reach, j);
        if (!seen) s4[r] = -INFINITY;
        // values that are not finite reach no row that does not see their key: they become 0, and
        // rows that do see it become NaN through their sum
        bool bad = false;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool off = !(__builtin_fabsf(now.v[r][n][c]) < INFINITY);
            bad = bad || off;
            if (off) now.v[r][n][c] = 0.f;
          }
        const uint64_t votes = __builtin_amdgcn_ballot_w64(bad);
        if (votes != 0 && seen && ((votes >> (16 * g)) & 0xffffu) != 0) total = NAN;
      }
    }
    const float m = across_rows(larger(larger(s4[0], s4[1]), larger(s4[2], s4[3])), larger);
    if (__builtin_amdgcn_ballot_w64(m > top) != 0) {
      const float next = larger(m, top);
      const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
      top = next;
      total *= f;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[n][c] *= f;
    }
    const float base = top == -INFINITY ? 0.f : top;
    float w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r] = __builtin_amdgcn_exp2f(s4[r] - base);
      total += w[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[n][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(now.v[r][n][c], w[r], acc[n][c], 0, 0, 0);
    if (!more) break;
#pragma unroll
    for (int s = 0; s < 4 * NB; ++s) now.k[s] = next.k[s];
    if (kBoth) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < NB; ++n) now.v[r][n] = next.v[r][n];
    }
    j0 = j1, end = end1, tile += kRowsWaves;
  }

  // the waves' sums: all to the largest top, then two and two
  total = across_rows(total, plus);
  if (g == 0) tops[wave][i] = top;
  __syncthreads();
  float best = tops[0][i];
#pragma unroll
  for (int w = 1; w < kRowsWaves; ++w) best = larger(best, tops[w][i]);
  const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - best);
  // a row whose total is NaN keeps it also where nothing else was seen
  total = total != total ? total : total * f;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[n][c] *= f;  // what is not finite stays so, however little it weighs
  if (g == 0) totals[wave][i] = total;
#pragma unroll
  for (int half = kRowsWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) share[((wave - half) * 4 * NB + n * 4 + c) * kWave + lane] = acc[n][c];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[n][c] += share[(wave * 4 * NB + n * 4 + c) * kWave + lane];
    }
    __syncthreads();
  }
  if (wave != 0 || !mine) return;
  total = totals[0][i];
#pragma unroll
  for (int w = 1; w < kRowsWaves; ++w) total += totals[w][i];
  if (splits == 1) {
    const bool empty = sees_nothing(reach);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        v4f o = {acc[n][0][rr], acc[n][1][rr], acc[n][2][rr], acc[n][3][rr]};
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = empty ? 0.f : o[c] / total;
        put4<VECTORS>(y + at, 64 * n + 16 * g + 4 * rr, p.dim, o);
      }
  } else {
    // [head][block][part][16] rows of 64 NB sums, then their tops and totals
    const uint64_t slot = ((static_cast<uint64_t>(head) * blocks + block) * splits + part) * kRowsBlock + i;
    const uint64_t slots = static_cast<uint64_t>(gridDim.x) * kRowsBlock;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const v4f o = {acc[n][0][rr], acc[n][1][rr], acc[n][2][rr], acc[n][3][rr]};
        put4<VECTORS>(sums + slot * (64 * NB), 64 * n + 16 * g + 4 * rr, p.dim, o);
      }
    if (g == 0) {
      sums[slots * (64 * NB) + 2 * slot] = best;
      sums[slots * (64 * NB) + 2 * slot + 1] = total;
    }
  }
}

// A wave a row: the parts' sums, all to the largest top.  Lane s has what part s needs, up to 64 parts, and four values of
// each part's sums.  A kernel of a few us is bound by fetching its code, so little is unrolled: 13 KB of it took
// 4.7 us for 32 rows of 16 parts, 3 KB take 3.9.
__global__ __launch_bounds__(kWave) void attention_join_kernel(const float* sums, float* y, uint32_t splits, uint32_t blocks,
                                                               uint32_t row_bits, uint32_t width, FastDiv f_rows,
                                                               uint32_t heads, AttentionArgs p) {
  constexpr int kTurn = 8;
  const uint32_t lane = threadIdx.x;
  const uint32_t block_rows = 1u << row_bits;
  uint32_t head, row, b, h, t, shared;
  fd_divmod(blockIdx.x, f_rows, head, row);
  fd_divmod(head, p.f_kv, b, h);
  fd_divmod(row, p.f_group, t, shared);
  const uint64_t slot = (static_cast<uint64_t>(head) * blocks + (row >> row_bits)) * splits * block_rows + (row & (block_rows - 1));
  const float* ends = sums + static_cast<uint64_t>(heads) * blocks * splits * block_rows * width;
  const float2 end = *reinterpret_cast<const float2*>(ends + 2 * (slot + min(lane, splits - 1) * block_rows));
  const float* from = sums + slot * width + min(4 * lane, width - 4);
  const uint32_t step = block_rows * width;
  v4f o[kTurn];
#pragma unroll
  for (int s = 0; s < kTurn; ++s) o[s] = *reinterpret_cast<const v4f*>(from + min(static_cast<uint32_t>(s), splits - 1) * step);
  asm volatile("" ::: "memory");
  const Sequence seq = sequence_of(p, b);
  if (static_cast<int>(t) >= seq.count) return;
  const bool empty = sees_nothing(reach_of(p, seq, t));
  const auto wave_join = [](float v, auto&& join) {
    v = join(v, dpp_f32<kDppXor1>(v));
    v = join(v, dpp_f32<kDppXor2>(v));
    v = join(v, dpp_f32<kDppHalfMirror>(v));
    v = join(v, dpp_f32<kDppMirror>(v));
    return across_rows(v, join);
  };
  const float top = lane < splits ? end.x : -INFINITY, best = wave_join(top, larger);
  const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - best);
  const float total = wave_join(lane >= splits ? 0.f : end.y != end.y ? end.y : end.y * f, plus);
  v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (uint32_t s0 = 0;;) {
#pragma unroll
    for (int s = 0; s < kTurn; ++s) {
      if (s0 + s >= splits) break;
      // a part that saw nothing holds zeros, one that saw something that is not finite counts with a weight of 0 as well
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s0 + s));
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(o[s][c], w, acc[c]);
    }
    s0 += kTurn;
    if (s0 >= splits) break;
#pragma unroll
    for (int s = 0; s < kTurn; ++s) o[s] = *reinterpret_cast<const v4f*>(from + min(s0 + s, splits - 1) * step);
  }
  float* yr = y + ((static_cast<uint64_t>(b) * p.length + t) * p.q_heads + h * p.group + shared) * p.dim;
  const int d = 4 * lane;
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = empty ? 0.f : acc[c] / total;
  if (d + 4 <= p.dim) *reinterpret_cast<v4f_unaligned*>(yr + d) = acc;
  else put4<false>(yr, d, p.dim, acc);
}

int join_parts(const float* sums, float* y, uint32_t splits, uint32_t blocks, uint32_t row_bits, uint32_t width, uint32_t heads,
               const AttentionArgs& p, hipStream_t st) {
  const uint32_t rows = static_cast<uint32_t>(p.length) * p.group;
  attention_join_kernel<<<heads * rows, kWave, 0, st>>>(sums, y, splits, blocks, row_bits, width, make_fastdiv(rows), heads, p);
  return launch_status();
}

// How many workgroups share the keys of a block of rows: as many as make the rounds of a workgroup for each compute unit
// short, none with fewer than four tiles, a wave each.  One round at a time is best: a sequence over 65536 keys of 8 heads 84 us in one
// round and 90 in two, 4 sequences of 4096 29 in one, 32 in two, 37 in four, 8 tokens over 4000 keys 21, 24, 33; 24 sequences,
// 192 blocks, 145 us with two parts and 124 with four, which are three whole rounds.
static int64_t rows_splits(int64_t items, int64_t tiles) {
  const int64_t units = 256, most = std::min<int64_t>({tiles / 4, 64, (units + items - 1) / items * 4});
  const auto rounds = [&](int64_t splits) { return (items * splits + units - 1) / units; };
  int64_t best = 1;
  for (int64_t splits = 2; splits <= most; ++splits)  // at least a twentieth shorter
    if (20 * rounds(splits) * best < 19 * rounds(best) * splits) best = splits;
  return best;
}
struct RowsPlan {
  uint32_t blocks, splits, groups;  // groups: workgroups of the grid
  size_t bytes;
};
static bool plan_rows(int batch, int length, int q_heads, int kv_heads, int dim, int capacity, int window, int sinks, int causal,
                      RowsPlan* plan) {
  const int64_t rows = static_cast<int64_t>(length) * (q_heads / kv_heads);
  const int64_t blocks = (rows + kRowsBlock - 1) / kRowsBlock, items = blocks * batch * kv_heads;
  const int64_t tiles = (most_keys(length, capacity, window, sinks, causal) + kRowsTile - 1) / kRowsTile;
  const int64_t splits = rows_splits(items, tiles);
  if (!grid_fits(items * splits, kRowsWaves * kWave)) return false;
  plan->blocks = static_cast<uint32_t>(blocks);
  plan->splits = static_cast<uint32_t>(splits);
  plan->groups = static_cast<uint32_t>(items * splits);
  const size_t width = static_cast<size_t>((dim + 63) / 64 * 64);
  plan->bytes = splits == 1 ? 0 : static_cast<size_t>(items * splits) * kRowsBlock * (width + 2) * sizeof(float);
  return true;
}

// Which kernel: from 65 rows of a key head on the keys and values are split for the 16-bit instructions first.  Over 4000 keys of
// 8 heads: 64 rows 31.5 us without that and 35.6 with, 96 rows 53.8 and 37.6; 16 sequences of 1900 keys of 64 values: 64 rows 45.1
// and 49.0, 96 rows 69.6 and 50.6.  So a token of 65 or more heads on one key head is split too: 128 heads of 64 over 8000 keys 23,
// of 128 over 65000 88.
static bool many_rows(int length, int q_heads, int kv_heads) {
  return static_cast<int64_t>(length) * (q_heads / kv_heads) > 64;
}

template <int NB, bool VECTORS>
static int launch_rows(const RowsPlan& plan, const float* q, const float* k, const float* v, float* y, float* sums, int batch,
                       const AttentionArgs& p, hipStream_t st) {
  attention_rows_kernel<NB, VECTORS><<<plan.groups, kRowsWaves * kWave, 0, st>>>(q, k, v, y, sums, make_fastdiv(plan.splits),
                                                                              make_fastdiv(plan.blocks), p);
  if (int rc = launch_status()) return rc;
  if (plan.splits == 1) return SHDW_OK;
  return join_parts(sums, y, plan.splits, plan.blocks, kRowsBits, 64 * NB, batch * p.kv_heads, p, st);
}

}  // namespace shdw

using namespace shdw;

namespace {

// What no call may have; everything else has a kernel.
int check_shape(int batch, int length, int q_heads, int kv_heads, int head_dim, int capacity, int window, int sinks) {
  if (batch < 0 || length < 0 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || capacity < 0 || window < 0 || sinks < 0)
    return SHDW_E_INVALID_ARGUMENT;
  if (q_heads % kv_heads != 0) return SHDW_E_INVALID_ARGUMENT;
  if (head_dim > kAttentionMaxDim) return SHDW_E_UNSUPPORTED;
  // rows and keys are counted in 32 bits, up to the ends of the last tiles
  const int64_t tokens = static_cast<int64_t>(batch) * length;
  if (capacity > kAttentionMost || tokens > kAttentionMost || tokens * q_heads > kAttentionMost) return SHDW_E_UNSUPPORTED;
  return SHDW_OK;
}

}  // namespace

extern "C" {

size_t shdw_hip_window_attention_workspace_bytes(int batch, int length, int q_heads, int kv_heads, int head_dim, int capacity,
                                                 int window, int sinks, int causal) {
  if (check_shape(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks) != SHDW_OK) return 0;
  if (batch == 0 || length == 0) return 0;
  if (many_rows(length, q_heads, kv_heads)) {
    TilesPlan plan;
    return plan_tiles(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks, causal, &plan) ? plan.bytes() : 0;
  }
  RowsPlan plan;
  return plan_rows(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks, causal, &plan) ? plan.bytes : 0;
}

int shdw_hip_window_attention(int batch, int length, int q_heads, int kv_heads, int head_dim, int capacity, int window, int sinks,
                              int causal, float scale, const float* q, const float* k, const float* v, const int* starts,
                              const int* lengths, float* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_shape(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks)) return rc;
  if (scale != scale) return SHDW_E_INVALID_ARGUMENT;
  if (batch == 0 || length == 0) return SHDW_OK;
  if (!q || !y || (capacity > 0 && (!k || !v)) || y == q || y == k || y == v) return SHDW_E_INVALID_ARGUMENT;
  AttentionArgs p;
  p.length = length, p.q_heads = q_heads, p.kv_heads = kv_heads, p.group = q_heads / kv_heads, p.dim = head_dim;
  p.capacity = capacity, p.window = window, p.sinks = sinks, p.causal = causal != 0;
  p.scale = scale, p.starts = starts, p.lengths = lengths;
  p.f_group = make_fastdiv(p.group), p.f_kv = make_fastdiv(kv_heads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto check_workspace = [&](size_t need) {
    if (need == 0) return SHDW_OK;
    if (!workspace || workspace_bytes < need) return SHDW_E_WORKSPACE;
    return aligned16(workspace) ? SHDW_OK : SHDW_E_INVALID_ARGUMENT;
  };
  if (many_rows(length, q_heads, kv_heads)) {
    TilesPlan plan;
    if (!plan_tiles(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks, causal, &plan)) return SHDW_E_UNSUPPORTED;
    if (int rc = check_workspace(plan.bytes())) return rc;
    return launch_tiles(plan, q, k, v, y, workspace, p, st);
  }
  RowsPlan plan;
  if (!plan_rows(batch, length, q_heads, kv_heads, head_dim, capacity, window, sinks, causal, &plan)) return SHDW_E_UNSUPPORTED;
  if (int rc = check_workspace(plan.bytes)) return rc;
  float* sums = static_cast<float*>(workspace);
  switch (head_dim < 4 ? 0 : (head_dim + 63) / 64) {
    case 0: return launch_rows<1, false>(plan, q, k, v, y, sums, batch, p, st);
    case 1: return launch_rows<1, true>(plan, q, k, v, y, sums, batch, p, st);
    case 2: return launch_rows<2, true>(plan, q, k, v, y, sums, batch, p, st);
    case 3: return launch_rows<3, true>(plan, q, k, v, y, sums, batch, p, st);
    default: return launch_rows<4, true>(plan, q, k, v, y, sums, batch, p, st);
  }
}

}  // extern "C"
