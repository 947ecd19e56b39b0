// Attention over a sliding window with first tokens that stay visible: backward pass.
//
//   p_ij  = exp(s_ij - lse_i)             dv_j = sum_i p_ij do_i
//   ds_ij = p_ij (do_i . v_j - delta_i)   delta_i = do_i . out_i
//   dq_i  = scale sum_j ds_ij k_j         dk_j = scale sum_i ds_ij q_i
//
// Two kernels, each of which owns what it sums: the first walks over the keys for a tile of rows (dq, and
// delta for the second), the second over the rows for a tile of keys (dk, dv).  The scores are formed
// twice, and sums that cross workgroups are added in a fixed order by a third kernel (chunk_plan):
// results do not depend on the order in which workgroups run.
//
// delta is taken from the output before its rounding (the forward pass keeps what the rounding left
// over): an error of delta is common to a whole row of ds, and with the rounded output it was the largest
// one in dq and dk (bf16, 512 tokens: 2.0e-3 of them against 1.7e-3 for rounding ds).  p and ds are rounded
// to the inputs' type, as operands of the matrix cores, and ds without scale, which the sums get in fp32.
// ds of fp16 inputs is multiplied by a power of two before it is rounded (kDsShift).  Rows that see a
// single key have zeros as ds by definition, not what p and delta's roundings would leave (dq: all such rows;
// dk: where all rows see few keys, so that nothing larger is added).
//
// Both kernels are built as the forward kernel is: a lane holds a row (first) or a key (second) of each
// result, which then is the next product's operand as it stands.  They are bound by the matrix cores, three
// and four products per tile, at the clock that their power leaves (1.7 to 2.0 GHz).  4 x 32 heads, 4096
// tokens, causal, 128 features, bf16: dq 0.81 to 0.86 ms and dk, dv 1.15 to 1.22 ms, 960 to 1020 and 900 to 960 TFLOP/s;
// window of 1024 over 2 x 8192 tokens, 32 heads on 8: 0.48 to 0.50 and 0.59 to 0.63 ms, 770 to 810 and 820 to 870
// TFLOP/s.  fp32, 777 patches: 50 to 53 and 57 to 62 us, 70 to 74 and 79 to 86 of the 139 TFLOP/s that a large product
// reaches.  (One launch that adds dq with atomics would save a product of the scores and lose the fixed order.)
#include <type_traits>

#include "attention.h"

namespace at_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kTileKeys = 32 * kWaves;   // keys that a workgroup of the second kernel owns
constexpr int kStep = 64;                // keys or rows of a tile it walks over

// WK waves share 32 rows and halve each tile of keys among them (1 or 2); they join at the end.
template <typename T, int DT, int WK>
__global__ __launch_bounds__(kWaves * 64, (kPerCu<T, DT>)) void attention_dq_kernel(AttentionArgs a) {
  typedef Tile<T, DT> L;
  typedef typename Frag<T>::type F;
  constexpr int kRows = 32 * kWaves / WK, kMine = kStep / WK;
  constexpr int kTileBytes = kStep * L::kPitch;
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
  const int head = h * a.group + g;

  F qf[L::kSteps], df[L::kSteps];
  float delta = 0.f;
  {
    const char* qp = a.q.p + b * a.q.batch + head * a.q.head + i * a.q.token;
    const char* dp = a.dout.p + b * a.dout.batch + head * a.dout.head + i * a.dout.token;
    const int64_t at = b * a.out.batch + head * a.out.head + i * a.out.token;
    const char *op = a.out.p + at, *rp = a.rest + at;
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) {
      const int d = s * 16 + half * 8;
      const bool in = valid && d < a.dim;
      qf[s] = in ? Frag<T>::load(qp + d * sizeof(T)) : Frag<T>::zero();
      df[s] = in ? Frag<T>::load(dp + d * sizeof(T)) : Frag<T>::zero();
      const F of = in ? Frag<T>::load(op + d * sizeof(T)) : Frag<T>::zero();
      float x[8], y[8];
      Frag<T>::unpack(df[s], x);
      Frag<T>::unpack(of, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
      if (sizeof(T) == 2 && a.rest) {
        Frag<T>::unpack(in ? Frag<T>::load(rp + d * sizeof(T)) : Frag<T>::zero(), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
      }
    }
  }
  delta = half_sum(delta);
  float lse = INFINITY;
  if (row < a.row_pitch) {
    lse = a.lse[(int64_t)bh * a.row_pitch + row];
    if (half == 0) a.delta[(int64_t)bh * a.row_pitch + row] = delta;
  }

  f32x16 dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dq[dt] = zero_acc();
  constexpr bool kFactor = ProbShift<T>::backward != 0.f;
  float base = (kFactor ? kDsShift : 0.f) - lse, undo = kFactor ? 1.f / kDsStart : 1.f;   // of the row's ds, see kDsShift

  const int p = seq.start + i;
  const int see_lo = valid ? p - a.left : 1, see_hi = valid ? min(p + a.right, seq.len - 1) : 0;
  const int see_sinks = valid ? min(a.sinks, a.causal ? p + 1 : seq.len) : 0;
  const int wrow0 = row0 + wave_row;
  const int first = seq.start + wrow0 / a.group;
  const int last = wrow0 < live_rows ? seq.start + (min(wrow0 + 32, live_rows) - 1) / a.group : first - 1;
  const KeyRange mine = keys_of(a, seq, first, last);

  int tiles = 0;
  KeyRange range = {0, 0, 0};
  if (row0 < live_rows)
    range = keys_of(a, seq, seq.start + row0 / a.group, seq.start + (min(row0 + kRows, live_rows) - 1) / a.group);
  const KeyWalk walk(range, max(a.k.token, a.v.token), kStep);
  if (row0 < live_rows) tiles = (walk.end + kStep - 1) / kStep;
  const char* kb = a.k.p + b * a.k.batch + h * a.k.head;
  const char* vb = a.v.p + b * a.v.batch + h * a.v.head;
  const int dim_bytes = a.dim * (int)sizeof(T);
  const int key_off = L::template lane_row<kWaves>() * (int)a.k.token, val_off = L::template lane_row<kWaves>() * (int)a.v.token;
  const int key_offs[2] = {L::template lane_offset<kWaves>(key_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(key_off, dim_bytes, 1)};
  const int val_offs[2] = {L::template lane_offset<kWaves>(val_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(val_off, dim_bytes, 1)};
  auto fetch = [&](int t, char* stage) {
    const int v0 = t * kStep, k0 = walk.first_key(v0);
    const i32x4 kr = open_rsrc(kb + k0 * a.k.token), vr = open_rsrc(vb + k0 * a.v.token);
    if (v0 >= walk.begin && v0 + kStep <= walk.end) {
      L::template fetch_all<kStep, kWaves>(kr, key_offs, kWaves * L::kLoadRows * (int)a.k.token, stage);
      L::template fetch_all<kStep, kWaves>(vr, val_offs, kWaves * L::kLoadRows * (int)a.v.token, stage + kTileBytes);
    } else {
      L::template fetch<kStep, kWaves>(kr, dim_bytes, stage, [&](int r) { return walk.offset(v0, r, (int)a.k.token); });
      L::template fetch<kStep, kWaves>(vr, dim_bytes, stage + kTileBytes,
                                      [&](int r) { return walk.offset(v0, r, (int)a.v.token); });
    }
  };

  if (tiles > 0) fetch(0, lds);
  // exact: ds goes into the product with what its rounding leaves over (see kFewKeys)
  auto go = [&](auto exact) {
    for (int t = 0; t < tiles; ++t) {
      char* stage = lds + (t & 1) * 2 * kTileBytes;
      lds_dma_wait_all();
      __syncthreads();
      if (t + 1 < tiles) fetch(t + 1, lds + ((t + 1) & 1) * 2 * kTileBytes);
      // the wave's part of the tile: places v0 ..; behind the sinks these are the keys k0 ..
      const int v0 = t * kStep + wave_key, k0 = v0 + walk.shift;
      const bool mixed = t * kStep < walk.begin;
      if (last < first || !(mixed || (k0 < mine.hi && k0 + kMine > mine.lo) || k0 < mine.sinks)) continue;
      const bool whole = !mixed && k0 >= last - a.left && k0 + kMine - 1 <= min(first + a.right, seq.len - 1);

      const typename L::Reader lr = L::reader(stage + wave_key * L::kPitch);
#pragma unroll
      for (int n = 0; n < kMine / 32; ++n) {
        f32x16 s = zero_acc(), dp = zero_acc();
#pragma unroll
        for (int ks = 0; ks < L::kSteps; ++ks) {
          Frag<T>::mma2(L::rows_frag(lr, 0, n * 32, ks), qf[ks], s, L::rows_frag(lr, kTileBytes, n * 32, ks), df[ks], dp);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, base)) * (dp[e] - delta);
        if (!whole) {
          int v = v0 + n * 32 + half * 4;
          asm volatile("" : "+v"(v));      // a branch: as selects the masks would be formed for every tile
          const int lo = max(see_lo - walk.shift, walk.begin) - v, hi = see_hi - walk.shift - v, sinks = see_sinks - v;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int c = acc_row(e, 0);
            s[e] = (c >= lo && c <= hi) || c < sinks ? s[e] : 0.f;
          }
        }
        if constexpr (kFactor) {
          const float top = largest(s);
          if (__any(top > kDsLimit)) {
            const DsFactor f = ds_factor(half_max(top));   // both halves of the wave add to a sum
            base += f.log2;
            undo *= inverse_power(f.value);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= f.value;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 16; ++e) dq[dt][e] *= f.value;
          }
        }
#pragma unroll
        for (int t16 = 0; t16 < 2; ++t16) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[t16 * 8 + e];
          const F ds = Frag<T>::pack(x);
          Frag<T>::mma_all([&](int dt) { return L::cols_frag(lr, 0, n * 32 + t16 * 16, dt); }, ds, dq);
          if constexpr (decltype(exact)::value)
            Frag<T>::mma_all([&](int dt) { return L::cols_frag(lr, 0, n * 32 + t16 * 16, dt); }, low_part<T>(x), dq);
        }
      }
    }
  };
  if constexpr (sizeof(T) == 2) {
    if (min(row0 + kRows, live_rows) <= rows_that_see(a, seq, kFewKeys)) go(std::true_type());
    else go(std::false_type());
  } else {
    go(std::false_type());
  }
  if constexpr (kFactor) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) dq[dt][e] *= undo;
  }

  if constexpr (WK > 1) {              // join the two halves of the keys
    typedef Exchange<16 * DT> X;
    static_assert(kWaves / 2 * X::kBytes <= (int)sizeof(lds), "the stages hold what is exchanged");
    char* room = lds + wave / 2 * X::kBytes;
    __syncthreads();                   // nobody reads the stages any more
    if (wave % 2 == 1) X::put(room, 0, dq);
    __syncthreads();
    if (wave % 2 == 1) return;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) dq[dt][e] += X::get(room, dt * 16 + e);
  }
  if (row >= all_rows) return;
  // the only key's probability is 1, whatever the query; and beside a padded row whole tiles were not masked
  if (!valid || row < rows_that_see(a, seq, 1)) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[dt] = zero_acc();
  }
  char* gp = a.dq.p + b * a.dq.batch + head * a.dq.head + i * a.dq.token;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = dt * 32 + q * 8 + half * 4;
      const float v[4] = {dq[dt][q * 4] * a.scale, dq[dt][q * 4 + 1] * a.scale, dq[dt][q * 4 + 2] * a.scale,
                          dq[dt][q * 4 + 3] * a.scale};
      if (d < a.dim) store_f32<T, 4>(reinterpret_cast<T*>(gp) + d, v);
    }
}

// The pieces of a head's dk and dv: `chunks` of every tile of keys, then `far_chunks` of the tiles with
// sinks (chunk_plan says why).
struct KeyPiece {
  int tile, chunk;
  bool far;
};
__host__ __device__ inline int key_pieces(const AttentionArgs& a) { return a.tiles * a.chunks + a.sink_tiles * a.far_chunks; }
__device__ __forceinline__ KeyPiece key_piece(const AttentionArgs& a, int rank) {
  const bool far = rank >= a.tiles * a.chunks;
  const int n = far ? rank - a.tiles * a.chunks : rank, per_tile = far ? a.far_chunks : a.chunks;
  return {n / per_tile, n % per_tile, far};
}

// Partial sums of a head: of every tile where all have several chunks, otherwise of the tiles with sinks.
// The place of a tile's first one (near chunks, then far ones), and for the last tile + 1 their number.
__host__ __device__ inline int64_t first_part(const AttentionArgs& a, int tile) {
  const int64_t sinks = tile < a.sink_tiles ? tile : a.sink_tiles;
  return sinks * (a.chunks + a.far_chunks) + (a.chunks > 1 ? (tile - sinks) * (int64_t)a.chunks : 0);
}

// Waves that share the walk over the rows that see nothing but the sinks of a tile: the tile's other keys
// must all lie within the near chunks, which start at the first row that sees the tile.  Not causal, that
// is the first row of all, and holds for the first tile only.
__host__ __device__ inline int sink_sharers(const AttentionArgs& a, int tile) {
  if (!a.causal && tile > 0) return 1;
  const int sinks = a.sinks - tile * kTileKeys;
  return sinks <= 32 ? 4 : sinks <= 64 ? 2 : 1;
}

// Steps of rows [begin, end) that see some key of a tile.
struct Steps {
  int begin, end;
};
__device__ __forceinline__ Steps steps_of(const AttentionArgs& a, const Sequence& s, int tile) {
  const int first = tile * kTileKeys, last = min(first + kTileKeys, s.len) - 1;
  const bool sinks = first < a.sinks;
  const int lo = !a.causal && sinks ? s.start : max(first - a.right, s.start);
  const int hi = sinks ? s.len - 1 : min(last + a.left, s.len - 1);
  if (first > last || lo > hi) return {0, 0};
  const int rows = min((hi - s.start + 1) * a.group, s.live * a.group);
  return {(lo - s.start) * a.group / kStep, (rows + kStep - 1) / kStep};
}

// The part of a tile's steps that a piece walks over.
__device__ __forceinline__ Steps steps_of(const AttentionArgs& a, const Steps& tile, int chunk, bool far) {
  const int length = far ? a.far_steps : a.chunk_steps;
  const int begin = tile.begin + (far ? a.chunks * a.chunk_steps : 0) + chunk * length;
  return {begin, min(tile.end, begin + length)};
}

// The step at which a piece begins its walk, which goes on to the end and then from the start.  The rows of
// a window are shifted from tile to tile by more than an L2 holds of all tiles' steps; begun at a multiple
// of the window's length, neighbours read the same rows at about the same time (window of 1024 over 8192
// tokens, 32 heads on 8: 2.42 -> 0.72 GiB from behind the L2, 625 -> 605 us; without a window nothing changes).
__device__ __forceinline__ int first_step(const AttentionArgs& a, const Steps& steps) {
  const int64_t period = ((int64_t)a.left + a.right + kTileKeys) * a.group / kStep;
  if (period > steps.end) return steps.begin;
  const int at = (steps.begin + (int)period - 1) / (int)period * (int)period;
  return at < steps.end ? at : steps.begin;
}

// Keys of a tile that far pieces have sums of.
__host__ __device__ inline int far_keys(const AttentionArgs& a, int tile) { return kTileKeys / sink_sharers(a, tile); }

__device__ __forceinline__ int wave_min(int v) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

// A wave owns 32 keys, whose keys and values stay in registers as operands, and walks over the rows that
// see them.  Of the rows that see sinks only, the waves of a workgroup share the walk instead: those with
// the same 32 keys take every second or fourth 32 rows (see chunk_plan for how the results are summed).
// EXACT: ds goes into the product with what its rounding leaves over (see kFewKeys), and is zero for rows that see
// a single key.
template <typename T, int DT, bool EXACT>
__global__ __launch_bounds__(kWaves * 64, (kPerCu<T, DT>)) void attention_dkv_kernel(AttentionArgs a) {
  typedef Tile<T, DT> L;
  typedef typename Frag<T>::type F;
  constexpr int kTileBytes = kStep * L::kPitch;
  constexpr int kStage = 2 * kTileBytes + 2048;                       // queries | output gradients | lse | delta
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // the first keys of a causal sequence are seen by the most rows; the short far pieces come last
  const Piece head_piece = piece_of(blockIdx.x, key_pieces(a), a.batch * a.kv_heads);
  const int bh = head_piece.bh;
  const KeyPiece piece = key_piece(a, head_piece.rank);
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const Sequence seq = sequence_of(a, b);
  const int live_rows = seq.live * a.group;
  const Steps steps = steps_of(a, steps_of(a, seq, piece.tile), piece.chunk, piece.far);
  const int begin = __builtin_amdgcn_readfirstlane(steps.begin), end = __builtin_amdgcn_readfirstlane(steps.end);
  if (begin >= end && (piece.far || a.chunks > 1)) return;    // no partial sum: the kernel that adds them knows
  // far from the tile's own tokens only its sinks are seen
  const int sharers = piece.far ? sink_sharers(a, piece.tile) : 1;
  const int subtile = wave % (kWaves / sharers), share = wave / (kWaves / sharers);
  const int key = piece.tile * kTileKeys + subtile * 32 + (lane & 31);
  int row_lo = 1 << 30, row_hi = -1;   // rows [row_lo, row_hi] see the key
  if (key < seq.len) {
    const bool sink = key < a.sinks;
    const int tok_lo = !a.causal && sink ? seq.start : max(key - a.right, seq.start);
    const int tok_hi = sink ? seq.len - 1 : min(key + a.left, seq.len - 1);
    if (tok_lo <= tok_hi) {
      row_lo = (tok_lo - seq.start) * a.group;
      row_hi = min((tok_hi - seq.start) * a.group + a.group, live_rows) - 1;
    }
  }
  F kf[L::kSteps], vf[L::kSteps];
  {
    const char* kp = a.k.p + b * a.k.batch + h * a.k.head + key * a.k.token;
    const char* vp = a.v.p + b * a.v.batch + h * a.v.head + key * a.v.token;
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) {
      const int d = s * 16 + half * 8;
      const bool in = row_hi >= 0 && d < a.dim;       // what nothing sees is not read
      kf[s] = in ? Frag<T>::load(kp + d * sizeof(T)) : Frag<T>::zero();
      vf[s] = in ? Frag<T>::load(vp + d * sizeof(T)) : Frag<T>::zero();
    }
  }
  // rows that some key of the wave, and that every key of it, is seen by
  const int any_lo = wave_min(row_lo), any_hi = -wave_min(-row_hi);
  const int all_lo = -wave_min(-row_lo), all_hi = wave_min(row_hi);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = zero_acc();
  constexpr bool kFactor = ProbShift<T>::backward != 0.f;
  float factor = kDsStart / 32768.f;   // of the key's ds beside the probabilities' own

  const char* qb = a.q.p + b * a.q.batch + (int64_t)h * a.group * a.q.head;
  const char* db = a.dout.p + b * a.dout.batch + (int64_t)h * a.group * a.dout.head;
  const float* lse = a.lse + (int64_t)bh * a.row_pitch;
  const float* delta = a.delta + (int64_t)bh * a.row_pitch;
  const int dim_bytes = a.dim * (int)sizeof(T);
  const float per_group = 1.f / (float)a.group;
  // rest + r is small, and the quotient's error far below the 0.5 / group that would change it
  auto offset = [&](int rest, int r, const Strided& x) {
    const int n = rest + r, token = (int)(((float)n + 0.5f) * per_group);
    return token * (int)x.token + (n - token * a.group) * (int)x.head;
  };
  // a group that divides the rows of a round: tiles and rounds start at a token's first head
  constexpr int kRound = kWaves * L::kLoadRows;
  const bool even = kRound % a.group == 0;
  const int q_off = offset(0, L::template lane_row<kWaves>(), a.q), d_off = offset(0, L::template lane_row<kWaves>(), a.dout);
  const int q_offs[2] = {L::template lane_offset<kWaves>(q_off, dim_bytes, 0),
                         L::template lane_offset<kWaves>(q_off, dim_bytes, 1)};
  const int d_offs[2] = {L::template lane_offset<kWaves>(d_off, dim_bytes, 0),
                         L::template lane_offset<kWaves>(d_off, dim_bytes, 1)};
  const int round_tokens = kRound / a.group;
  auto fetch = [&](int t, char* stage) {
    const int r0 = t * kStep;
    const int i0 = r0 / a.group, rest = r0 - i0 * a.group;
    const i32x4 qr = open_rsrc(qb + i0 * a.q.token), dr = open_rsrc(db + i0 * a.dout.token);
    if (even && r0 + kStep <= live_rows) {
      L::template fetch_all<kStep, kWaves>(qr, q_offs, round_tokens * (int)a.q.token, stage);
      L::template fetch_all<kStep, kWaves>(dr, d_offs, round_tokens * (int)a.dout.token, stage + kTileBytes);
    } else {
      L::template fetch<kStep, kWaves>(qr, dim_bytes, stage,
                                       [&](int r) { return r0 + r < live_rows ? offset(rest, r, a.q) : -1; });
      L::template fetch<kStep, kWaves>(dr, dim_bytes, stage + kTileBytes,
                                       [&](int r) { return r0 + r < live_rows ? offset(rest, r, a.dout) : -1; });
    }
    if (wave < 2)   // 64 values each: lanes 0..15 move 16 bytes, the others write zeros behind them
      dma_16(open_rsrc((const char*)((wave == 0 ? lse : delta) + r0)), lane < 16 ? lane * 16 : kOobOffset, 0,
             stage + 2 * kTileBytes + wave * 1024);
  };

  const int start = __builtin_amdgcn_readfirstlane(first_step(a, steps)), count = end - begin;
  const int single = __builtin_amdgcn_readfirstlane(rows_that_see(a, seq, 1));
  if (count > 0) fetch(start, lds);
  for (int u = 0, t = start, next; u < count; ++u, t = next) {
    char* stage = lds + (u & 1) * kStage;
    next = t + 1 < end ? t + 1 : begin;
    lds_dma_wait_all();
    __syncthreads();
    if (u + 1 < count) fetch(next, lds + ((u + 1) & 1) * kStage);
    const typename L::Reader lr = L::reader(stage);
    const float* stats = reinterpret_cast<const float*>(stage + 2 * kTileBytes);
#pragma unroll
    for (int n = 0; n < kStep / 32; ++n) {
      const int r0 = t * kStep + n * 32;
      if (r0 > any_hi || r0 + 31 < any_lo || ((t * (kStep / 32) + n) & (sharers - 1)) != share) continue;
      const bool whole = r0 >= all_lo && r0 + 31 <= all_hi;
      f32x16 s = zero_acc(), dp = zero_acc();
#pragma unroll
      for (int ks = 0; ks < L::kSteps; ++ks) {
        Frag<T>::mma2(L::rows_frag(lr, 0, n * 32, ks), kf[ks], s, L::rows_frag(lr, kTileBytes, n * 32, ks), vf[ks], dp);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 l4 = *reinterpret_cast<const float4*>(stats + n * 32 + q * 8 + half * 4);
        const float4 d4 = *reinterpret_cast<const float4*>(stats + 256 + n * 32 + q * 8 + half * 4);
        const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, de[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = q * 4 + j;
          s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, ProbShift<T>::backward - ls[j]));
          dp[e] = s[e] * (dp[e] - de[j]);
        }
      }
      if (!whole) {
        int row = r0 + half * 4;
        asm volatile("" : "+v"(row));    // a branch: as selects the masks would be formed for every tile
        const int lo = row_lo - row, hi = row_hi - row;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool seen = acc_row(e, 0) >= lo && acc_row(e, 0) <= hi;
          s[e] = seen ? s[e] : 0.f;
          dp[e] = seen ? dp[e] : 0.f;
        }
        if (EXACT && r0 < single) {      // probabilities of 1, whatever the key
#pragma unroll
          for (int e = 0; e < 16; ++e) dp[e] = row + acc_row(e, 0) < single ? 0.f : dp[e];
        }
      }
      if constexpr (kFactor) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] *= factor;
        const float top = largest(dp);
        if (__any(top > kDsLimit)) {
          const DsFactor f = ds_factor(half_max(top));   // both halves of the wave add to a sum
          factor *= f.value;
#pragma unroll
          for (int e = 0; e < 16; ++e) dp[e] *= f.value;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) dk[dt][e] *= f.value;
        }
      }
#pragma unroll
      for (int t16 = 0; t16 < 2; ++t16) {
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = s[t16 * 8 + e];
          y[e] = dp[t16 * 8 + e];
        }
        const F pf = Frag<T>::pack(x), df = Frag<T>::pack(y);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          Frag<T>::mma2(L::cols_frag(lr, kTileBytes, n * 32 + t16 * 16, dt), pf, dv[dt],
                        L::cols_frag(lr, 0, n * 32 + t16 * 16, dt), df, dk[dt]);
        }
        if constexpr (EXACT && sizeof(T) == 2)
          Frag<T>::mma_all([&](int dt) { return L::cols_frag(lr, 0, n * 32 + t16 * 16, dt); }, low_part<T>(y), dk);
      }
    }
  }

  const float dv_scale = kFactor ? 1.f / 32768.f : 1.f;
  if constexpr (kFactor) {
    const float undo = dv_scale * inverse_power(factor);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[dt][e] *= undo;
  }

  if (sharers > 1) {                   // the first wave of each 32 keys takes the others' sums over
    typedef Exchange<32 * DT> X;
    static_assert(2 * X::kBytes <= (int)sizeof(lds), "the stages hold what is exchanged");
    for (int n = kWaves / 2; n >= kWaves / sharers; n /= 2) {
      __syncthreads();                 // nobody reads the stages, or what was exchanged, any more
      if (wave >= n && wave < 2 * n) {
        X::put(lds + (wave - n) * X::kBytes, 0, dk);
        X::put(lds + (wave - n) * X::kBytes, 16 * DT, dv);
      }
      __syncthreads();
      if (wave < n) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            dk[dt][e] += X::get(lds + wave * X::kBytes, dt * 16 + e);
            dv[dt][e] += X::get(lds + wave * X::kBytes, (DT + dt) * 16 + e);
          }
      }
    }
    if (share > 0) return;
  }

  const bool seen = row_lo <= row_hi;  // otherwise the sums hold 0 times rows, NaN where these are not finite
  const bool partial = a.chunks > 1 || (piece.tile < a.sink_tiles && subtile * 32 < far_keys(a, piece.tile));
  float* part = a.part + (int64_t)(wave * 32 + (lane & 31)) * a.dim +
                (bh * first_part(a, a.tiles) + first_part(a, piece.tile) + (piece.far ? a.chunks : 0) + piece.chunk) *
                    (2 * kTileKeys * a.dim);
  char* kp = a.dk.p + b * a.dk.batch + h * a.dk.head + key * a.dk.token;
  char* vp = a.dv.p + b * a.dv.batch + h * a.dv.head + key * a.dv.token;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = dt * 32 + q * 8 + half * 4;
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = seen ? dk[dt][q * 4 + j] * a.scale : 0.f;
        y[j] = seen ? dv[dt][q * 4 + j] * dv_scale : 0.f;
      }
      if (d >= a.dim) continue;
      if (partial) {                   // one of several partial sums
        store_f32<float, 4>(part + d, x);
        store_f32<float, 4>(part + kTileKeys * a.dim + d, y);
      } else if (key < a.keys) {
        store_f32<T, 4>(reinterpret_cast<T*>(kp) + d, x);
        store_f32<T, 4>(reinterpret_cast<T*>(vp) + d, y);
      }
    }
}

// Sums the partial dk and dv of a key, in a fixed order.  32 lanes cover dim with four elements each.  A
// workgroup of 8 such groups takes GROUPS of them for a key: one where all keys have a few sums, all 8
// where only the sinks have any, and many.
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(AttentionArgs a) {
  __shared__ float4 sums[2][8][32];
  const unsigned tiles = a.chunks > 1 ? a.tiles : a.sink_tiles;
  const unsigned at = blockIdx.x * (8 / GROUPS) + (GROUPS == 1 ? threadIdx.x >> 5 : 0);
  const int bh = (int)(at / (tiles * kTileKeys)), rest = (int)(at - bh * tiles * kTileKeys);
  const int tile = rest / kTileKeys, local = rest % kTileKeys;
  const int key = tile * kTileKeys + local, group = GROUPS == 1 ? 0 : threadIdx.x >> 5, d = (threadIdx.x & 31) * 4;
  const bool sinks = tile < a.sink_tiles && local < far_keys(a, tile);
  if (key >= a.keys || (a.chunks == 1 && !sinks)) return;     // written by the only piece that has it
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  // the sums that were written: pieces without rows wrote none
  const Steps steps = steps_of(a, sequence_of(a, b), tile);
  const int count = max(steps.end - steps.begin, 0);
  const int near = a.chunks == 1 ? 1 : min(a.chunks, (count + a.chunk_steps - 1) / a.chunk_steps);
  const int beyond = count - a.chunks * a.chunk_steps;
  const int far = sinks && beyond > 0 ? min(a.far_chunks, (beyond + a.far_steps - 1) / a.far_steps) : 0;
  const int64_t next = 2LL * kTileKeys * a.dim;
  const float* part = a.part + (bh * first_part(a, a.tiles) + first_part(a, tile)) * next + (int64_t)local * a.dim + d;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
  if (d < a.dim) {
#pragma unroll 4
    for (int n = group; n < near + far; n += GROUPS) {
      const float* p = part + (n < near ? n : a.chunks + n - near) * next;
      float u[4], w[4];
      load_f32<float, 4>(p, u);
      load_f32<float, 4>(p + (int64_t)kTileKeys * a.dim, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] += u[j];
        y[j] += w[j];
      }
    }
  }
  T* const to_k = reinterpret_cast<T*>(a.dk.p + b * a.dk.batch + h * a.dk.head + key * a.dk.token) + d;
  T* const to_v = reinterpret_cast<T*>(a.dv.p + b * a.dv.batch + h * a.dv.head + key * a.dv.token) + d;
  if constexpr (GROUPS == 1) {
    if (d < a.dim) {
      store_f32<T, 4>(to_k, x);
      store_f32<T, 4>(to_v, y);
    }
  } else {
    sums[0][group][threadIdx.x & 31] = make_float4(x[0], x[1], x[2], x[3]);
    sums[1][group][threadIdx.x & 31] = make_float4(y[0], y[1], y[2], y[3]);
    __syncthreads();
    if (group > 1 || d >= a.dim) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float4 u = sums[group][n][threadIdx.x & 31];
      v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
    }
    store_f32<T, 4>(group == 0 ? to_k : to_v, v);
  }
}

// How dk and dv are cut up.  The rows that see a tile of keys are walked over in steps of 64.  Where the
// tiles alone do not give every CU two workgroups, the steps of each are cut into chunks, whose partial sums
// another kernel adds.  With a window a tile is seen by few rows, but a tile with sinks by all of them: the
// rows beyond the others' reach are far pieces of their own, short ones that fill up the end of the launch
// (window 1024 over 8192 tokens, bf16: one workgroup per head for all rows of the sinks 5.1 ms).
void chunk_plan(AttentionArgs& a) {
  a.tiles = (int)cdiv64(a.keys, kTileKeys);
  const int64_t heads = (int64_t)a.batch * a.kv_heads, rows = (int64_t)a.rows * a.group;
  const int64_t near = (int64_t)(a.left + a.right + kTileKeys) * a.group;
  const int64_t span = near < rows ? near : rows;              // rows that see a tile without sinks
  const int64_t want = a.slots;
  int64_t steps = cdiv64(span, kStep) + 1;                     // the first step need not start at the first row
  a.chunks = 1;
  if (a.tiles * heads > 0 && a.tiles * heads < want && steps > 2) {
    // on average, half of the chunks of a causal sequence without a window have no rows
    const int64_t groups = a.causal && span == rows ? cdiv64(a.tiles * heads, 2) : a.tiles * heads;
    int64_t n = (want + groups / 2) / groups;
    if (n > steps / 2) n = steps / 2;
    a.chunks = (int)n;
    steps = cdiv64(steps, n);
  }
  a.chunk_steps = (int)steps;
  const int64_t far = cdiv64(rows, kStep) + 1 - steps * a.chunks;
  a.sink_tiles = a.sinks > 0 && far > 0 && heads > 0 ? (int)cdiv64(a.sinks, kTileKeys) : 0;   // no heads: an empty batch
  a.far_chunks = a.far_steps = 0;
  if (a.sink_tiles > 0) {
    int64_t n = cdiv64(want, a.sink_tiles * heads);
    if (n > cdiv64(far, 8)) n = cdiv64(far, 8);
    a.far_steps = (int)cdiv64(far, n);
    a.far_chunks = (int)cdiv64(far, a.far_steps);
  }
}

int64_t delta_bytes(const AttentionArgs& a) { return (int64_t)a.batch * a.kv_heads * a.row_pitch * 4; }

int64_t part_bytes(const AttentionArgs& a) {
  return (int64_t)a.batch * a.kv_heads * first_part(a, a.tiles) * 2 * kTileKeys * a.dim * 4;
}

template <typename T, int DT>
int launch(AttentionArgs a, hipStream_t stream) {
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  chunk_plan(a);
  const int64_t pieces = key_pieces(a) * heads;
  const int64_t joined = (int64_t)(a.chunks > 1 ? a.tiles : a.sink_tiles) * kTileKeys * heads;
  const int64_t rows = (int64_t)a.rows * a.group;
  const bool share = waves_per_row(rows, heads, a.slots) == 2;
  const int64_t row_tiles = cdiv64(rows, share ? 64 : 128);
  if (!grid_fits(row_tiles * heads) || !grid_fits(pieces) || !grid_fits(joined)) return AT_ERR_DIM;
  int rc = AT_OK;
  if (a.rows > 0) {
    AttentionArgs r = a;
    r.tiles = (int)row_tiles;
    const dim3 grid((unsigned)(row_tiles * heads)), block(kWaves * 64);
    if (share) hipLaunchKernelGGL((attention_dq_kernel<T, DT, 2>), grid, block, 0, stream, r);
    else hipLaunchKernelGGL((attention_dq_kernel<T, DT, 1>), grid, block, 0, stream, r);
    rc = launch_status();
    if (rc != AT_OK) return rc;
  }
  // kernels of their own: with both in one the registers do not suffice
  if (a.keys <= kFewKeys || a.left + a.right + a.sinks < kFewKeys)
    hipLaunchKernelGGL((attention_dkv_kernel<T, DT, true>), dim3((unsigned)pieces), dim3(kWaves * 64), 0, stream, a);
  else
    hipLaunchKernelGGL((attention_dkv_kernel<T, DT, false>), dim3((unsigned)pieces), dim3(kWaves * 64), 0, stream, a);
  rc = launch_status();
  if (rc != AT_OK || joined == 0) return rc;
  if (a.chunks > 1)                    // whole tiles of keys: a multiple of 8 of them
    hipLaunchKernelGGL((attention_dkv_join_kernel<T, 1>), dim3((unsigned)(joined / 8)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attention_dkv_join_kernel<T, 8>), dim3((unsigned)joined), dim3(256), 0, stream, a);
  return launch_status();
}

template <typename T>
int launch_dim(const AttentionArgs& a, hipStream_t stream) {
  switch ((a.dim + 31) / 32) {
    case 1: return launch<T, 1>(a, stream);
    case 2: return launch<T, 2>(a, stream);
    case 3: return launch<T, 3>(a, stream);
    default: return launch<T, 4>(a, stream);
  }
}

}  // namespace
}  // namespace at_hip

using namespace at_hip;

extern "C" {

int64_t at_attention_bwd_workspace_bytes(const at_attention_t* shape) {
  AttentionArgs a;
  if (attention_args(shape, a) != AT_OK || a.batch == 0 || a.keys == 0) return 0;
  chunk_plan(a);
  return delta_bytes(a) + part_bytes(a);
}

int at_attention_bwd(const at_attention_t* shape, const void* output_grad, const void* q, const void* k, const void* v,
                     const void* lengths, const void* query_lengths, const void* out, const void* out_rest,
                     const float* lse, void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes, at_stream_t stream) {
  AttentionArgs a;
  const int rc = attention_args(shape, a);
  if (rc != AT_OK) return rc;
  if (a.batch == 0 || a.keys == 0) return AT_OK;
  if (!k || !v || !dk || !dv || (a.rows > 0 && (!output_grad || !q || !out || !lse || !dq))) return AT_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(output_grad) || !aligned16(dq) ||
      !aligned16(dk) || !aligned16(dv) || !aligned16(lse) || !aligned16(workspace) || !aligned16(out_rest))
    return AT_ERR_ALIGN;
  const int64_t need = at_attention_bwd_workspace_bytes(shape);
  if (need > 0 && (!workspace || workspace_bytes < need)) return AT_ERR_WORKSPACE;
  a.q.p = (char*)q; a.k.p = (char*)k; a.v.p = (char*)v; a.out.p = (char*)out; a.dout.p = (char*)output_grad;
  a.dq.p = (char*)dq; a.dk.p = (char*)dk; a.dv.p = (char*)dv;
  a.rest = (char*)out_rest;
  a.lengths = lengths;
  a.query_lengths = query_lengths;
  a.lse = const_cast<float*>(lse);
  a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(a));   // row_pitch keeps it on 256 bytes
  if (shape->dtype == AT_DTYPE_F32) return launch_dim<float>(a, (hipStream_t)stream);
  if (shape->dtype == AT_DTYPE_F16) return launch_dim<f16_t>(a, (hipStream_t)stream);
  return launch_dim<bf16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
