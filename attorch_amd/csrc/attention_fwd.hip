// Attention over a sliding window with first tokens that stay visible: forward pass.
//
//   s_ij = scale q_i . k_j over the visible j,   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// in one pass over the keys: the running maximum m_i and the running sum are kept per row, and what
// was summed before is rescaled when the maximum grows (exponentials in base 2, fp32 throughout).  The
// probabilities are rounded to the inputs' type for the second product only, since the matrix cores take
// 16-bit operands of one type: 2^-9 (bf16) or 2^-12 (fp16) of each on average, as much again as rounding
// the output leaves (bf16: 2.3e-3 of the output's norm with both, 1.7e-3 with the output's alone).  Where
// rows see few keys, what that rounding leaves over takes part in a product of its own (kFewKeys).
//
// The product is formed as keys x rows, so that a lane holds one row: the maximum and the sum need one
// exchange between the two halves of a wave, and the probabilities leave the matrix cores as the second
// product's operand.  Four waves of 32 rows each walk over tiles of 64 keys, which are loaded to LDS
// without passing through registers, one tile ahead; the keys and values that the waves share are read
// once, and two workgroups per CU let one's exponentials run under the other's products.
//
// Many rows: bound by the matrix cores and the exponentials, 16 of which take as long as half of the 16
// products of a 32 x 32 tile of 128 features, and by the power of both: the clock falls to 1.75 GHz.  4 x 32
// heads, 4096 tokens, causal, 128 features, bf16: 0.68 to 0.72 ms, 770 to 810 TFLOP/s; window of 1024 over 2 x
// 8192 tokens, 32 heads on 8: 0.36 to 0.38 ms, 680 to 715 TFLOP/s; a chunk of 1024 tokens over 16384 with a window of
// 4096: 87 to 91 us, 750 to 790 TFLOP/s.  fp32, 777 patches: 37 us, 66 TFLOP/s.
// Single tokens: bound by reading the keys and values once.  64 conversations of 4096 to 8192 tokens, 32
// heads on 8, bf16: 319 us, 5.0 TB/s; one of 131072: 97 us and 6 us for the join, 5.4 TB/s.  (Tiles of 32
// keys with up to five on their way read 4.5 TB/s: fewer, larger loads keep memory busier.  For many rows
// they leave room for three workgroups per CU: window 1024 358 -> 341 us, but 346 -> 360 us for causal
// rows of 64 features and 70 -> 84 us for fewer workgroups than that fills.)
#include <algorithm>
#include <type_traits>

#include "attention.h"

namespace at_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxSplits = 128;

// Four elements of the output, and what their rounding left over where a backward pass will need it.
template <typename T>
__device__ __forceinline__ void store_output(const AttentionArgs& a, int64_t to, const float (&v)[4]) {
  store_f32<T, 4>(reinterpret_cast<T*>(a.out.p + to), v);
  if constexpr (sizeof(T) == 2) {
    if (a.rest) {
      float r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = v[j] - to_f32(from_f32<T>(v[j]));
      store_f32<T, 4>(reinterpret_cast<T*>(a.rest + to), r);
    }
  }
}

// WK waves share 32 rows and halve each tile of KEYS keys among them (1 or 2); they join at the end.
template <typename T, int DT, int WK, int KEYS>
__global__ __launch_bounds__(kWaves * 64, (KEYS == 32 ? 2 : kPerCu<T, DT>)) void attention_fwd_kernel(AttentionArgs a) {
  typedef Tile<T, DT> L;
  typedef typename Frag<T>::type F;
  constexpr int kTileBytes = KEYS * L::kPitch;
  constexpr int kRows = 32 * kWaves / WK, kMine = KEYS / WK, NS = kMine / 32;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];   // two stages of keys | values

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Piece piece = piece_of(blockIdx.x, a.tiles, a.batch * a.kv_heads);
  const int tile_id = a.tiles - 1 - piece.rank;    // the last rows of a causal sequence see the most keys
  const int bh = piece.bh;
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const Sequence seq = sequence_of(a, b);
  const int live_rows = seq.live * a.group, all_rows = a.rows * a.group;
  const int row0 = tile_id * kRows;

  const int wave_row = wave / WK * 32, wave_key = wave % WK * kMine;
  const int row = row0 + wave_row + (lane & 31);
  const int i = row / a.group, g = row - i * a.group;
  const bool valid = row < live_rows;

  F qf[L::kSteps];
  {
    const char* qp = a.q.p + b * a.q.batch + (int64_t)(h * a.group + g) * a.q.head + i * a.q.token;
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) {
      const int d = s * 16 + half * 8;
      qf[s] = valid && d < a.dim ? Frag<T>::load(qp + d * sizeof(T)) : Frag<T>::zero();
    }
  }
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = zero_acc();
  float m = -INFINITY, l = 0.f;

  // what this lane's row sees
  const int p = seq.start + i;
  const int see_lo = valid ? p - a.left : 1, see_hi = valid ? min(p + a.right, seq.len - 1) : 0;
  const int see_sinks = valid ? min(a.sinks, a.causal ? p + 1 : seq.len) : 0;
  // tokens of the wave's rows (last < first: none is live)
  const int wrow0 = row0 + wave_row;
  const int first = seq.start + wrow0 / a.group;
  const int last = wrow0 < live_rows ? seq.start + (min(wrow0 + 32, live_rows) - 1) / a.group : first - 1;
  const KeyRange mine = keys_of(a, seq, first, last);

  int tiles = 0;
  KeyRange range = {0, 0, 0};
  if (row0 < live_rows)
    range = keys_of(a, seq, seq.start + row0 / a.group, seq.start + (min(row0 + kRows, live_rows) - 1) / a.group);
  const KeyWalk walk(range, max(a.k.token, a.v.token), KEYS);
  if (row0 < live_rows) tiles = (walk.end + KEYS - 1) / KEYS;
  const int split = blockIdx.y;
  const int t_begin = (int)((int64_t)tiles * split / a.splits), t_end = (int)((int64_t)tiles * (split + 1) / a.splits);

  const char* kb = a.k.p + b * a.k.batch + h * a.k.head;
  const char* vb = a.v.p + b * a.v.batch + h * a.v.head;
  const int dim_bytes = a.dim * (int)sizeof(T);
  const int key_off = L::template lane_row<kWaves>() * (int)a.k.token, val_off = L::template lane_row<kWaves>() * (int)a.v.token;
  const int key_offs[2] = {L::template lane_offset<kWaves>(key_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(key_off, dim_bytes, 1)};
  const int val_offs[2] = {L::template lane_offset<kWaves>(val_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(val_off, dim_bytes, 1)};
  auto fetch = [&](int t, char* stage) {
    const int v0 = t * KEYS, k0 = walk.first_key(v0);
    const i32x4 kr = open_rsrc(kb + k0 * a.k.token), vr = open_rsrc(vb + k0 * a.v.token);
    if (v0 >= walk.begin && v0 + KEYS <= walk.end) {
      L::template fetch_all<KEYS, kWaves>(kr, key_offs, kWaves * L::kLoadRows * (int)a.k.token, stage);
      L::template fetch_all<KEYS, kWaves>(vr, val_offs, kWaves * L::kLoadRows * (int)a.v.token, stage + kTileBytes);
    } else {
      L::template fetch<KEYS, kWaves>(kr, dim_bytes, stage, [&](int r) { return walk.offset(v0, r, (int)a.k.token); });
      L::template fetch<KEYS, kWaves>(vr, dim_bytes, stage + kTileBytes,
                                      [&](int r) { return walk.offset(v0, r, (int)a.v.token); });
    }
  };

  if (t_begin < t_end) fetch(t_begin, lds);
  // exact: the second product takes what the rounding of the probabilities leaves over as well (see kFewKeys)
  auto walk_keys = [&](auto exact) {
    for (int t = t_begin; t < t_end; ++t) {
      char* stage = lds + ((t - t_begin) & 1) * 2 * kTileBytes;
      lds_dma_wait_all();
      __syncthreads();     // tile t is everybody's, and nobody reads the other stage any more
      if (t + 1 < t_end) fetch(t + 1, lds + ((t - t_begin + 1) & 1) * 2 * kTileBytes);
      // the wave's part of the tile: places v0 ..; behind the sinks these are the keys k0 ..
      const int v0 = t * KEYS + wave_key, k0 = v0 + walk.shift;
      const bool mixed = t * KEYS < walk.begin;
      if (last < first || !(mixed || (k0 < mine.hi && k0 + kMine > mine.lo) || k0 < mine.sinks)) continue;

      const typename L::Reader lr = L::reader(stage + wave_key * L::kPitch);
      f32x16 s[NS];
#pragma unroll
      for (int n = 0; n < NS; ++n) s[n] = zero_acc();
#pragma unroll
      for (int ks = 0; ks < L::kSteps; ++ks)
        Frag<T>::mma_all([&](int n) { return L::rows_frag(lr, 0, n * 32, ks); }, qf[ks], s);
      // places of the lane relative to its first one are constants: 8 apart, 4 in a row
      const bool whole = !mixed && k0 >= last - a.left && k0 + kMine - 1 <= min(first + a.right, seq.len - 1);
      if (!whole) {
        int v = v0 + half * 4;
        asm volatile("" : "+v"(v));      // a branch: as selects the masks would be formed for every tile
        const int lo = max(see_lo - walk.shift, walk.begin) - v, hi = see_hi - walk.shift - v, sinks = see_sinks - v;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int c = n * 32 + acc_row(e, 0);
            s[n][e] = (c >= lo && c <= hi) || c < sinks ? s[n][e] : -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(fmaxf(top, s[0][e]), s[NS - 1][e]);
      top = half_max(top) * a.scale_log2;
      // The exponentials are taken relative to a maximum that may lag behind by kSlack: any reference gives
      // the same result, and moving it costs a pass over the output, which now is rare.
      if (__any(top > m + kSlack)) {
        const float old = m;
        m = fmaxf(m, top);
        const float shrink = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(old - m);
        l *= shrink;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= shrink;
      }
      const float base = m == -INFINITY ? 0.f : ProbShift<T>::forward - m;   // -inf: the row has seen nothing yet
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[n][e] = __builtin_amdgcn_exp2f(fmaf(s[n][e], a.scale_log2, base));
          sum[e & 3] += s[n][e];
        }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int ks = 0; ks < kMine / 16; ++ks) {
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) pr[e] = s[ks >> 1][(ks & 1) * 8 + e];
        const F pf = Frag<T>::pack(pr);
        Frag<T>::mma_all([&](int dt) { return L::cols_frag(lr, kTileBytes, ks * 16, dt); }, pf, o);
        if constexpr (decltype(exact)::value)
          Frag<T>::mma_all([&](int dt) { return L::cols_frag(lr, kTileBytes, ks * 16, dt); }, low_part<T>(pr), o);
      }
    }
  };
  if constexpr (sizeof(T) == 2) {
    if (min(row0 + kRows, live_rows) <= rows_that_see(a, seq, kFewKeys)) walk_keys(std::true_type());
    else walk_keys(std::false_type());
  } else {
    walk_keys(std::false_type());
  }

  l = half_sum(l);
  if constexpr (WK > 1) {              // join the two halves of the keys
    typedef Exchange<16 * DT + 2> X;
    static_assert(kWaves / 2 * X::kBytes <= (int)sizeof(lds), "the stages hold what is exchanged");
    char* room = lds + wave / 2 * X::kBytes;
    __syncthreads();                   // nobody reads the stages any more
    if (wave % 2 == 1) {
      X::put(room, 2, o);
      reinterpret_cast<float*>(room)[lane] = m;
      reinterpret_cast<float*>(room)[64 + lane] = l;
    }
    __syncthreads();
    if (wave % 2 == 1) return;
    const float m1 = X::get(room, 0), l1 = X::get(room, 1), top = fmaxf(m, m1);
    const float w0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float w1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - top);
    m = top;
    l = l * w0 + l1 * w1;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * w0 + X::get(room, 2 + dt * 16 + e) * w1;
  }
  if (!valid) {          // a padded row, beside which whole tiles were not masked: anything, NaN where keys are not finite
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = zero_acc();
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  const float lse = valid ? m + __builtin_amdgcn_logf(l) - ProbShift<T>::forward : INFINITY;
  if (a.splits > 1) {
    if (row >= all_rows) return;
    float* part = a.part + (((int64_t)split * a.batch * a.kv_heads + bh) * all_rows + row) * a.dim;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = dt * 32 + q * 8 + half * 4;
        if (d < a.dim)
          *reinterpret_cast<float4*>(part + d) = make_float4(o[dt][q * 4] * inv, o[dt][q * 4 + 1] * inv,
                                                             o[dt][q * 4 + 2] * inv, o[dt][q * 4 + 3] * inv);
      }
    if (half == 0)
      a.part_lse[((int64_t)split * a.batch * a.kv_heads + bh) * a.row_pitch + row] = l == 0.f ? -INFINITY : lse;
    return;
  }
  if (a.lse && half == 0 && row < a.row_pitch) a.lse[(int64_t)bh * a.row_pitch + row] = lse;
  if (row >= all_rows) return;
  const int64_t to = b * a.out.batch + (int64_t)(h * a.group + g) * a.out.head + i * a.out.token;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = dt * 32 + q * 8 + half * 4;
      const float v[4] = {o[dt][q * 4] * inv, o[dt][q * 4 + 1] * inv, o[dt][q * 4 + 2] * inv, o[dt][q * 4 + 3] * inv};
      if (d < a.dim) store_output<T>(a, to + d * (int)sizeof(T), v);
    }
}

// Joins the splits of a row: out = sum_s 2^(lse_s - lse) out_s, lse = log2 sum_s 2^lse_s.  32 lanes cover
// dim with four elements each.  A workgroup of 8 such groups takes GROUPS of them for a row: one where the
// splits are few (then bound by reading them: 33 MB in 10 us), all 8 where they are many, each on every
// eighth split (one group over 64 splits: 51 us for one token of 131072, eight: 4).
constexpr int kFewSplits = 8;
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
  __shared__ float4 sums[8][32];
  const int all_rows = a.rows * a.group;
  const int64_t bhs = (int64_t)a.batch * a.kv_heads;
  const int64_t at = (int64_t)blockIdx.x * (8 / GROUPS) + (GROUPS == 1 ? threadIdx.x >> 5 : 0);
  if (at >= bhs * all_rows) return;
  const int bh = (int)(at / all_rows), row = (int)(at - (int64_t)bh * all_rows);
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int i = row / a.group, g = row - i * a.group;
  const int first = GROUPS == 1 ? 0 : threadIdx.x >> 5, d = (threadIdx.x & 31) * 4;
  const bool valid = i < sequence_of(a, b).live;

  const float* lses = a.part_lse + (int64_t)bh * a.row_pitch + row;
  const int64_t next = bhs * a.row_pitch;
  float top = -INFINITY, total = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  __shared__ float shared_lse[GROUPS == 1 ? 1 : kMaxSplits];
  if constexpr (GROUPS == 1) {
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, lses[s * next]);
  } else {                             // one round of loads for all splits
    for (int s = threadIdx.x; s < a.splits; s += 256) shared_lse[s] = lses[s * next];
    __syncthreads();
    for (int s = threadIdx.x & 63; s < a.splits; s += 64) top = fmaxf(top, shared_lse[s]);
    top = wave_reduce(top, kWave, MaxOp());
  }
  if (top == -INFINITY) top = 0.f;
#pragma unroll 4
  for (int s = first; s < a.splits; s += GROUPS) {
    const float w = __builtin_amdgcn_exp2f((GROUPS == 1 ? lses[s * next] : shared_lse[s]) - top);
    total += w;
    if (d < a.dim) {
      const float4 x = *reinterpret_cast<const float4*>(a.part + ((s * bhs + bh) * all_rows + row) * a.dim + d);
      v[0] += w * x.x; v[1] += w * x.y; v[2] += w * x.z; v[3] += w * x.w;
    }
  }
  if constexpr (GROUPS > 1) {
    __shared__ float totals[8];
    sums[first][threadIdx.x & 31] = make_float4(v[0], v[1], v[2], v[3]);
    if ((threadIdx.x & 31) == 0) totals[first] = total;
    __syncthreads();
    if (first != 0) return;
#pragma unroll
    for (int n = 1; n < GROUPS; ++n) {
      const float4 x = sums[n][threadIdx.x];
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      total += totals[n];
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = valid ? v[j] * inv : 0.f;
  if (d < a.dim)
    store_output<T>(a, b * a.out.batch + (int64_t)(h * a.group + g) * a.out.head + i * a.out.token + d * (int)sizeof(T), v);
  if (!a.lse) return;
  float* lse = a.lse + (int64_t)bh * a.row_pitch;
  if (d == 0) lse[row] = valid ? top + __builtin_amdgcn_logf(total) : INFINITY;
  if (row == all_rows - 1)             // and the padding behind the last row
    for (int r = all_rows + (threadIdx.x & 31); r < a.row_pitch; r += 32) lse[r] = INFINITY;
}

// How the work is cut: into tiles of 128 rows, or of 64 whose waves share rows in pairs (waves_per_row), and
// where these do not fill the GPU, the keys are split among several workgroups with at least four tiles of
// keys each, which another launch of 4 us joins (a tile takes a workgroup about 1).
//
// fp32 heads of more than 64 features fill LDS with one workgroup's tiles of 64 keys.  Tiles of 32 let a CU
// hold two workgroups, which pays where there are several for each place, and for single tokens where the
// splits fill them all: window of 512 over 4096 tokens, 32 heads on 8 of 128: 344 -> 287 us; single tokens
// over 64 x 600: 198 -> 102 us, 16 x 4096: 201 -> 172 us, 32768: 97 -> 89 us.  Elsewhere waves that share
// rows, or workgroups that follow each other, do better: causal, 2 x 2048 tokens, 16 heads: 307 against 372
// us; single tokens over 5 x 2359, 4 heads: 37 against 50 us.
void plan(AttentionArgs& a) {
  const int64_t heads = (int64_t)a.batch * a.kv_heads, rows = (int64_t)a.rows * a.group;
  // keys that one tile of rows can see
  auto tiles_seen = [&](int64_t tile_rows) {
    const int64_t span = (int64_t)a.left + a.right + cdiv64(tile_rows, a.group) + a.sinks;
    return cdiv64(span < a.keys ? span : a.keys, 64);
  };
  const int64_t two_per_cu = 2 * (int64_t)device_cu_count();
  const int64_t whole = cdiv64(rows, 32 * kWaves) * heads;
  a.narrow = a.slots < two_per_cu &&
             (whole >= 2 * two_per_cu || (rows <= 32 && heads * std::max<int64_t>(tiles_seen(32 * kWaves) / 4, 1) >= two_per_cu));
  const int64_t want = a.narrow ? two_per_cu : a.slots;
  a.waves_per_row = a.narrow ? 1 : waves_per_row(rows, heads, a.slots);
  const int64_t tile_rows = 32 * kWaves / a.waves_per_row;
  a.tiles = (int)cdiv64(rows, tile_rows);
  a.splits = 1;
  const int64_t groups = a.tiles * heads;
  if (groups >= want || groups == 0) return;
  const int64_t tiles = tiles_seen(tile_rows);
  int64_t n = want / groups;           // rounded up, a few workgroups would run after all the others
  if (n > tiles / 4) n = tiles / 4;
  a.splits = (int)(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
}

template <typename T, int DT>
void launch(const AttentionArgs& a, const dim3& grid, hipStream_t stream) {
  const dim3 block(kWaves * 64);
  if constexpr (kPerCu<T, DT> == 1) {
    if (a.narrow) {
      hipLaunchKernelGGL((attention_fwd_kernel<T, DT, 1, 32>), grid, block, 0, stream, a);
      return;
    }
  }
  if (a.waves_per_row == 1) hipLaunchKernelGGL((attention_fwd_kernel<T, DT, 1, 64>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attention_fwd_kernel<T, DT, 2, 64>), grid, block, 0, stream, a);
}

template <typename T>
int launch_dim(const AttentionArgs& a, hipStream_t stream) {
  const int64_t blocks = (int64_t)a.tiles * a.batch * a.kv_heads;
  const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows * a.group;
  if (!grid_fits(blocks) || (a.splits > 1 && !grid_fits(rows))) return AT_ERR_DIM;
  const dim3 grid((unsigned)blocks, (unsigned)a.splits);
  switch ((a.dim + 31) / 32) {
    case 1: launch<T, 1>(a, grid, stream); break;
    case 2: launch<T, 2>(a, grid, stream); break;
    case 3: launch<T, 3>(a, grid, stream); break;
    default: launch<T, 4>(a, grid, stream); break;
  }
  int rc = launch_status();
  if (rc == AT_OK && a.splits > 1) {
    if (a.splits <= kFewSplits)
      hipLaunchKernelGGL((attention_join_kernel<T, 1>), dim3((unsigned)cdiv64(rows, 8)), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((attention_join_kernel<T, 8>), dim3((unsigned)rows), dim3(256), 0, stream, a);
    rc = launch_status();
  }
  return rc;
}

int64_t part_bytes(const AttentionArgs& a) {
  if (a.splits <= 1) return 0;
  return (int64_t)a.splits * a.batch * a.kv_heads * ((int64_t)a.rows * a.group * a.dim + a.row_pitch) * 4;
}

}  // namespace
}  // namespace at_hip

using namespace at_hip;

extern "C" {

int64_t at_attention_row_pitch(int64_t rows, int64_t heads, int64_t kv_heads) {
  if (rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return 0;
  return cdiv64(rows * (heads / kv_heads), kRowAlign) * kRowAlign;
}

int64_t at_attention_fwd_workspace_bytes(const at_attention_t* shape) {
  AttentionArgs a;
  if (attention_args(shape, a) != AT_OK) return 0;
  plan(a);
  return part_bytes(a);
}

int at_attention_fwd(const at_attention_t* shape, const void* q, const void* k, const void* v,
                     const void* lengths, const void* query_lengths, void* out, float* lse, void* out_rest,
                     void* workspace, int64_t workspace_bytes, at_stream_t stream) {
  AttentionArgs a;
  const int rc = attention_args(shape, a);
  if (rc != AT_OK) return rc;
  if (a.batch == 0 || a.rows == 0) return AT_OK;
  if (!q || !out || (a.keys > 0 && (!k || !v))) return AT_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(lse) || !aligned16(out_rest) ||
      !aligned16(workspace))
    return AT_ERR_ALIGN;
  a.q.p = (char*)q; a.k.p = (char*)k; a.v.p = (char*)v; a.out.p = (char*)out;
  a.lengths = lengths;
  a.query_lengths = query_lengths;
  a.lse = lse;
  a.rest = (char*)out_rest;
  plan(a);
  const int64_t need = part_bytes(a);
  if (need > 0 && (!workspace || workspace_bytes < need)) return AT_ERR_WORKSPACE;
  a.part = (float*)workspace;
  a.part_lse = a.splits > 1 ? a.part + (int64_t)a.splits * a.batch * a.kv_heads * a.rows * a.group * a.dim : nullptr;
  if (shape->dtype == AT_DTYPE_F32) return launch_dim<float>(a, (hipStream_t)stream);
  if (shape->dtype == AT_DTYPE_F16) return launch_dim<f16_t>(a, (hipStream_t)stream);
  return launch_dim<bf16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
