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
// one in dq and dk (bf16, 512 tokens: 2.0e-3 of them against 1.7e-3 for rounding ds).
#include "attention.h"

namespace at_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kStep = 64;                // keys or rows of a tile it walks over

// WK waves share 32 rows and halve each tile of keys among them (1 or 2); they join at the end.
template <typename T, int DT, int WK>
__global__ __launch_bounds__(kWaves * 64, sizeof(T) == 2 ? 2 : 1) void attention_dq_kernel(AttentionArgs a) {
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

  const int p = seq.start + i;
  const int see_lo = valid ? p - a.left : 1, see_hi = valid ? min(p + a.right, seq.len - 1) : 0;
  const int see_sinks = valid ? min(a.sinks, a.causal ? p + 1 : seq.len) : 0;
  const int wrow0 = row0 + wave_row;
  const int first = seq.start + wrow0 / a.group;
  const int last = wrow0 < live_rows ? seq.start + (min(wrow0 + 32, live_rows) - 1) / a.group : first - 1;
  const KeyRange mine = keys_of(a, seq, first, last);

  int tiles_lo = 0, sink_tiles = 0, tiles = 0;
  KeyRange range = {0, 0, 0};
  if (row0 < live_rows) {
    range = keys_of(a, seq, seq.start + row0 / a.group, seq.start + (min(row0 + kRows, live_rows) - 1) / a.group);
    tiles_lo = range.lo / kStep;
    sink_tiles = min((range.sinks + kStep - 1) / kStep, tiles_lo);
    tiles = sink_tiles + (max(range.hi, range.sinks) + kStep - 1) / kStep - tiles_lo;
  }
  const char* kb = a.k.p + b * a.k.batch + h * a.k.head;
  const char* vb = a.v.p + b * a.v.batch + h * a.v.head;
  const int dim_bytes = a.dim * (int)sizeof(T);
  auto first_key = [&](int t) { return (t < sink_tiles ? t : t - sink_tiles + tiles_lo) * kStep; };
  const int key_off = L::template lane_row<kWaves>() * (int)a.k.token, val_off = L::template lane_row<kWaves>() * (int)a.v.token;
  const int key_offs[2] = {L::template lane_offset<kWaves>(key_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(key_off, dim_bytes, 1)};
  const int val_offs[2] = {L::template lane_offset<kWaves>(val_off, dim_bytes, 0),
                           L::template lane_offset<kWaves>(val_off, dim_bytes, 1)};
  auto fetch = [&](int t, char* stage) {
    const int k0 = first_key(t);
    const i32x4 kr = open_rsrc(kb + k0 * a.k.token), vr = open_rsrc(vb + k0 * a.v.token);
    if (k0 >= range.lo && k0 + kStep <= range.hi) {
      L::template fetch_all<kStep, kWaves>(kr, key_offs, kWaves * L::kLoadRows * (int)a.k.token, stage);
      L::template fetch_all<kStep, kWaves>(vr, val_offs, kWaves * L::kLoadRows * (int)a.v.token, stage + kTileBytes);
    } else {
      L::template fetch<kStep, kWaves>(kr, dim_bytes, stage, [&](int r) { return range.has(k0 + r) ? r * (int)a.k.token : -1; });
      L::template fetch<kStep, kWaves>(vr, dim_bytes, stage + kTileBytes,
                                      [&](int r) { return range.has(k0 + r) ? r * (int)a.v.token : -1; });
    }
  };

  if (tiles > 0) fetch(0, lds);
  for (int t = 0; t < tiles; ++t) {
    char* stage = lds + (t & 1) * 2 * kTileBytes;
    lds_dma_wait_all();
    __syncthreads();
    if (t + 1 < tiles) fetch(t + 1, lds + ((t + 1) & 1) * 2 * kTileBytes);
    const int k0 = first_key(t) + wave_key;
    if (!((k0 < mine.hi && k0 + kMine > mine.lo) || k0 < mine.sinks) || last < first) continue;
    const bool whole = k0 >= last - a.left && k0 + kMine - 1 <= min(first + a.right, seq.len - 1);

    const typename L::Reader lr = L::reader(stage + wave_key * L::kPitch);
#pragma unroll
    for (int n = 0; n < kMine / 32; ++n) {
      f32x16 s = zero_acc(), dp = zero_acc();
#pragma unroll
      for (int ks = 0; ks < L::kSteps; ++ks) {
        s = Frag<T>::mma(L::rows_frag(lr, 0, n * 32, ks), qf[ks], s);
        dp = Frag<T>::mma(L::rows_frag(lr, kTileBytes, n * 32, ks), df[ks], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -lse)) * (dp[e] - delta);
      if (!whole) {
        int key = k0 + n * 32 + half * 4;
        asm volatile("" : "+v"(key));    // a branch: as selects the masks would be formed for every tile
        const int lo = see_lo - key, hi = see_hi - key, sinks = see_sinks - key;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = acc_row(e, 0);
          s[e] = (c >= lo && c <= hi) || c < sinks ? s[e] : 0.f;
        }
      }
#pragma unroll
      for (int t16 = 0; t16 < 2; ++t16) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[t16 * 8 + e];
        const F ds = Frag<T>::pack(x);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          dq[dt] = Frag<T>::mma(L::cols_frag(lr, 0, n * 32 + t16 * 16, dt), ds, dq[dt]);
      }
    }
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

// Work items of a head whose results are partial sums, and the number of item `nth` of its class among them.
__host__ __device__ inline int64_t part_items(const AttentionArgs& a) {
  return (int64_t)(a.sink_chunks > 1 ? a.sink_tiles * a.sink_chunks : 0) +
         (a.chunks > 1 ? (int64_t)(a.tiles - a.sink_tiles) * a.chunks : 0);
}
__host__ __device__ inline int64_t part_item(const AttentionArgs& a, bool of_sinks, int nth) {
  return of_sinks || a.sink_chunks <= 1 ? nth : (int64_t)a.sink_tiles * a.sink_chunks + nth;
}

__device__ __forceinline__ int wave_min(int v) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

// A wave owns KT x 32 keys: their keys and values stay in registers as operands, and every fragment of
// queries and output gradients that it reads from LDS serves KT products.
template <typename T, int DT, int KT>
__global__ __launch_bounds__(kWaves * 64, KT == 1 && sizeof(T) == 2 ? 2 : 1) void attention_dkv_kernel(AttentionArgs a) {
  typedef Tile<T, DT> L;
  typedef typename Frag<T>::type F;
  constexpr int kTileBytes = kStep * L::kPitch;
  constexpr int kStage = 2 * kTileBytes + 2048;                       // queries | output gradients | lse | delta
  constexpr int kTileKeys = 32 * KT * kWaves;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // the first keys of a causal sequence are seen by the most rows
  const Piece piece = piece_of(blockIdx.x, a.sink_tiles * a.sink_chunks + (a.tiles - a.sink_tiles) * a.chunks,
                               a.batch * a.kv_heads);
  const int item = piece.rank, bh = piece.bh;
  const bool of_sinks = item < a.sink_tiles * a.sink_chunks;
  const int nth = of_sinks ? item : item - a.sink_tiles * a.sink_chunks;
  const int tile_chunks = of_sinks ? a.sink_chunks : a.chunks;
  const int chunk = nth % tile_chunks;
  const int tile_id = nth / tile_chunks + (of_sinks ? 0 : a.sink_tiles);
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const Sequence seq = sequence_of(a, b);
  const int live_rows = seq.live * a.group;
  const int key0 = tile_id * kTileKeys + wave * 32 * KT + (lane & 31);   // this lane's keys: key0 + 32 kt

  F kf[KT][L::kSteps], vf[KT][L::kSteps];
  int row_lo[KT], row_hi[KT];          // rows [row_lo, row_hi] see the key
  int any_lo = 1 << 30, any_hi = -1, all_lo = 0, all_hi = 1 << 30;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int key = key0 + 32 * kt;
    const bool valid = key < seq.len;
    const char* kp = a.k.p + b * a.k.batch + h * a.k.head + key * a.k.token;
    const char* vp = a.v.p + b * a.v.batch + h * a.v.head + key * a.v.token;
    row_lo[kt] = 1 << 30;
    row_hi[kt] = -1;
    if (valid) {
      const bool sink = key < a.sinks;
      const int tok_lo = !a.causal && sink ? seq.start : max(key - a.right, seq.start);
      const int tok_hi = sink ? seq.len - 1 : min(key + a.left, seq.len - 1);
      if (tok_lo <= tok_hi) {
        row_lo[kt] = (tok_lo - seq.start) * a.group;
        row_hi[kt] = min((tok_hi - seq.start) * a.group + a.group, live_rows) - 1;
      }
    }
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) {
      const int d = s * 16 + half * 8;
      const bool in = row_hi[kt] >= 0 && d < a.dim;       // what nothing sees is not read
      kf[kt][s] = in ? Frag<T>::load(kp + d * sizeof(T)) : Frag<T>::zero();
      vf[kt][s] = in ? Frag<T>::load(vp + d * sizeof(T)) : Frag<T>::zero();
    }
    any_lo = min(any_lo, row_lo[kt]);
    any_hi = max(any_hi, row_hi[kt]);
    all_lo = max(all_lo, row_lo[kt]);
    all_hi = min(all_hi, row_hi[kt]);
  }
  // rows that some key of the wave, and that every key of it, is seen by
  any_lo = wave_min(any_lo);
  any_hi = -wave_min(-any_hi);
  all_lo = -wave_min(-all_lo);
  all_hi = wave_min(all_hi);
  f32x16 dk[KT][DT], dv[KT][DT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[kt][dt] = dv[kt][dt] = zero_acc();

  __shared__ int ranges[2 * kWaves];
  if (lane == 0) {
    ranges[wave] = any_lo;
    ranges[kWaves + wave] = any_hi;
  }
  __syncthreads();
  int begin = ranges[0], end = ranges[kWaves];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    begin = min(begin, ranges[w]);
    end = max(end, ranges[kWaves + w]);
  }
  begin = begin / kStep + chunk * a.chunk_steps;
  end = min(end < 0 ? 0 : end / kStep + 1, begin + a.chunk_steps);
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);

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

  if (begin < end) fetch(begin, lds);
  for (int t = begin; t < end; ++t) {
    char* stage = lds + ((t - begin) & 1) * kStage;
    lds_dma_wait_all();
    __syncthreads();
    if (t + 1 < end) fetch(t + 1, lds + ((t + 1 - begin) & 1) * kStage);
    const typename L::Reader lr = L::reader(stage);
    const float* stats = reinterpret_cast<const float*>(stage + 2 * kTileBytes);
#pragma unroll
    for (int n = 0; n < kStep / 32; ++n) {
      const int r0 = t * kStep + n * 32;
      if (r0 > any_hi || r0 + 31 < any_lo) continue;
      const bool whole = r0 >= all_lo && r0 + 31 <= all_hi;
      f32x16 s[KT], dp[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = dp[kt] = zero_acc();
#pragma unroll
      for (int ks = 0; ks < L::kSteps; ++ks) {
        const F qf = L::rows_frag(lr, 0, n * 32, ks), df = L::rows_frag(lr, kTileBytes, n * 32, ks);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          s[kt] = Frag<T>::mma(qf, kf[kt][ks], s[kt]);
          dp[kt] = Frag<T>::mma(df, vf[kt][ks], dp[kt]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 l4 = *reinterpret_cast<const float4*>(stats + n * 32 + q * 8 + half * 4);
        const float4 d4 = *reinterpret_cast<const float4*>(stats + 256 + n * 32 + q * 8 + half * 4);
        const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, de[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int e = q * 4 + j;
            s[kt][e] = __builtin_amdgcn_exp2f(fmaf(s[kt][e], a.scale_log2, ProbShift<T>::backward - ls[j]));
            dp[kt][e] = s[kt][e] * (dp[kt][e] - de[j]);
          }
      }
      if (!whole) {
        int row = r0 + half * 4;
        asm volatile("" : "+v"(row));    // a branch: as selects the masks would be formed for every tile
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int lo = row_lo[kt] - row, hi = row_hi[kt] - row;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool seen = acc_row(e, 0) >= lo && acc_row(e, 0) <= hi;
            s[kt][e] = seen ? s[kt][e] : 0.f;
            dp[kt][e] = seen ? dp[kt][e] : 0.f;
          }
        }
      }
#pragma unroll
      for (int t16 = 0; t16 < 2; ++t16) {
        F pf[KT], df[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          float x[8], y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = s[kt][t16 * 8 + e];
            y[e] = dp[kt][t16 * 8 + e];
            if (ProbShift<T>::backward != 0.f) y[e] *= 1.f / 32768.f;
          }
          pf[kt] = Frag<T>::pack(x);
          df[kt] = Frag<T>::pack(y);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const F dc = L::cols_frag(lr, kTileBytes, n * 32 + t16 * 16, dt);
          const F qc = L::cols_frag(lr, 0, n * 32 + t16 * 16, dt);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            dv[kt][dt] = Frag<T>::mma(dc, pf[kt], dv[kt][dt]);
            dk[kt][dt] = Frag<T>::mma(qc, df[kt], dk[kt][dt]);
          }
        }
      }
    }
  }

  const float dv_scale = ProbShift<T>::backward != 0.f ? 1.f / 32768.f : 1.f;
  float* part = a.part + ((int64_t)bh * part_items(a) + part_item(a, of_sinks, nth)) * 2 * kTileKeys * a.dim +
                (int64_t)(wave * 32 * KT + (lane & 31)) * a.dim;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int key = key0 + 32 * kt;
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
          x[j] = dk[kt][dt][q * 4 + j] * a.scale;
          y[j] = dv[kt][dt][q * 4 + j] * dv_scale;
        }
        if (d >= a.dim) continue;
        if (tile_chunks > 1) {         // one of several partial sums
          store_f32<float, 4>(part + kt * 32 * a.dim + d, x);
          store_f32<float, 4>(part + (kTileKeys + kt * 32) * a.dim + d, y);
        } else if (key < a.keys) {
          store_f32<T, 4>(reinterpret_cast<T*>(kp) + d, x);
          store_f32<T, 4>(reinterpret_cast<T*>(vp) + d, y);
        }
      }
  }
}

// Sums the partial dk and dv of the tiles that were worked on in chunks, in the chunks' order.  32 lanes per
// key, four elements of dim per lane.
template <typename T, int kTileKeys>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(AttentionArgs a) {
  const int first_tile = a.sink_chunks > 1 ? 0 : a.sink_tiles;
  const int tiles = (a.chunks > 1 ? a.tiles : a.sink_tiles) - first_tile;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int bh = (int)(at / ((int64_t)tiles * kTileKeys));
  if (bh >= a.batch * a.kv_heads) return;
  const int rest = (int)(at - (int64_t)bh * tiles * kTileKeys);
  const int tile = first_tile + rest / kTileKeys, local = rest % kTileKeys;
  const int key = tile * kTileKeys + local, d = (threadIdx.x & 31) * 4;
  if (key >= a.keys || d >= a.dim) return;
  const bool of_sinks = tile < a.sink_tiles;
  const int chunks = of_sinks ? a.sink_chunks : a.chunks;
  const int nth = of_sinks ? tile * chunks : (tile - a.sink_tiles) * chunks;
  const float* part = a.part + (((int64_t)bh * part_items(a) + part_item(a, of_sinks, nth)) * 2 * kTileKeys + local) * a.dim + d;
  const int64_t other = (int64_t)kTileKeys * a.dim;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = 0; c < chunks; ++c) {
    float u[4], w[4];
    load_f32<float, 4>(part + c * 2 * other, u);
    load_f32<float, 4>(part + c * 2 * other + other, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] += u[j];
      y[j] += w[j];
    }
  }
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  store_f32<T, 4>(reinterpret_cast<T*>(a.dk.p + b * a.dk.batch + h * a.dk.head + key * a.dk.token) + d, x);
  store_f32<T, 4>(reinterpret_cast<T*>(a.dv.p + b * a.dv.batch + h * a.dv.head + key * a.dv.token) + d, y);
}

#ifndef KTSEL
#define KTSEL 32
#endif
constexpr int keys_per_wave(int dtype, int dim_tiles) { return dtype == AT_DTYPE_F32 ? 32 : KTSEL; }
template <typename T, int DT> constexpr int keys_per_wave() { return keys_per_wave(dtype_of<T>::value, DT); }

// How dk and dv are cut up.  The rows that see a tile of keys are walked over in chunks of chunk_steps
// steps; tiles with one chunk write their result, the others partial sums that a second kernel adds.
// With a window a tile is seen by few rows, but a tile with sinks by all: such tiles are cut to the
// others' length, or one workgroup per head would run on alone (window 1024 over 8192 tokens: 5.1 ms
// instead of 1.3).  Where the tiles alone do not give every CU two workgroups, all are cut further.
void chunk_plan(AttentionArgs& a, int tile_keys) {
  a.tile_keys = tile_keys;
  a.tiles = (int)cdiv64(a.keys, tile_keys);
  const int64_t rows = (int64_t)a.rows * a.group;
  const int64_t near = (int64_t)(a.left + a.right + tile_keys) * a.group;
  const int64_t span = near < rows ? near : rows;              // of a tile without sinks
  a.sink_tiles = span < rows ? (int)cdiv64(a.sinks, tile_keys) : 0;
  int64_t steps = cdiv64(span, kStep) + 1;                     // the first step need not start at the first row
  const int64_t groups = (int64_t)a.tiles * a.batch * a.kv_heads;
  const int64_t want = 2 * device_cu_count();
  if (groups < want && steps > 2) {
    int64_t n = cdiv64(want, groups);
    if (n > steps / 2) n = steps / 2;
    steps = cdiv64(steps, n);
  }
  a.chunk_steps = (int)steps;
  a.chunks = (int)cdiv64(cdiv64(span, kStep) + 1, steps);
  a.sink_chunks = (int)cdiv64(cdiv64(rows, kStep) + 1, steps);
}

int64_t delta_bytes(const AttentionArgs& a) { return (int64_t)a.batch * a.kv_heads * a.row_pitch * 4; }

int64_t part_bytes(const AttentionArgs& a) {
  return (int64_t)a.batch * a.kv_heads * part_items(a) * 2 * a.tile_keys * a.dim * 4;
}

template <typename T, int DT>
int launch(AttentionArgs a, hipStream_t stream) {
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  constexpr int KT = keys_per_wave<T, DT>() / 32;
  chunk_plan(a, kWaves * 32 * KT);
  const int64_t items = (int64_t)a.sink_tiles * a.sink_chunks + (int64_t)(a.tiles - a.sink_tiles) * a.chunks;
  // tiles of 128 rows, or of 64 where these give no more than two workgroups per CU: see the forward pass
  const int64_t rows = (int64_t)a.rows * a.group;
  const bool share = cdiv64(rows, 32 * kWaves) * heads < 2 * device_cu_count();
  const int64_t row_tiles = cdiv64(rows, 32 * kWaves / (share ? 2 : 1));
  const int64_t joined = ((a.chunks > 1 ? a.tiles : a.sink_tiles) - (a.sink_chunks > 1 ? 0 : a.sink_tiles)) *
                         (int64_t)a.tile_keys * heads;
  if (!grid_fits(row_tiles * heads) || !grid_fits(items * heads) || !grid_fits(cdiv64(joined, 8))) return AT_ERR_DIM;
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
  hipLaunchKernelGGL((attention_dkv_kernel<T, DT, KT>), dim3((unsigned)(items * heads)), dim3(kWaves * 64), 0, stream, a);
  rc = launch_status();
  if (rc != AT_OK || part_items(a) == 0) return rc;
  hipLaunchKernelGGL((attention_dkv_join_kernel<T, kWaves * 32 * KT>), dim3((unsigned)cdiv64(joined, 8)), dim3(256), 0, stream, a);
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
  if (attention_args(shape, a) != AT_OK || a.keys == 0) return 0;
  chunk_plan(a, kWaves * keys_per_wave(shape->dtype, (a.dim + 31) / 32));
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
