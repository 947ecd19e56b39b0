// Building blocks shared by the attention kernels: arguments, the visibility rule, LDS tiles and
// matrix-core fragments.
//
// Rows.  The query heads that share a key head are folded into one list of rows: row r of a
// key head is token r / group of query head r % group.  The rows of a tile then span few
// tokens, so a window or a causal edge wastes little of a tile, and one pass over the keys
// serves every query head that shares them.
//
// Visibility.  A sequence has `len` tokens; its first row is token `start`, and `live` rows are
// tokens of it (the others are padding).  Row of token p sees key j < len when j lies in
// [p - left, p + right] or j is one of the first `sinks` (and j <= p where causal).
#pragma once

#include "at_mfma.h"

namespace at_hip {

// Workgroups of four waves that a CU holds: two, but for the wide tiles of fp32.
template <typename T, int DT> constexpr int kPerCu = sizeof(T) == 4 && DT > 2 ? 1 : 2;

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kFar = 1 << 30;          // more than any distance between two tokens

struct Strided {                       // [batch, head, token, dim] tensor; strides in bytes
  char* p;
  int64_t batch, head, token;
};

struct AttentionArgs {
  Strided q, k, v, out, dout, dq, dk, dv;
  char* rest;                          // nullable; out before its rounding minus out, in out's layout and type
  float* lse;                          // [batch * kv_heads][row_pitch]: log2 of the row's sum of exponentials
  float* delta;                        // backward, same layout: sum over dim of output * output_grad
  float* part;                         // forward in splits: unreduced outputs [split][batch * kv_heads][rows][dim], fp32
  float* part_lse;                     // and their log2 sums [split][batch * kv_heads][row_pitch]
  const void* lengths;                 // tokens of each sequence, or null: `keys` of all
  const void* query_lengths;           // live rows of each sequence, or null: `rows` of all
  int lengths64, causal;
  int batch, kv_heads, group, rows, keys, dim;
  int row_pitch, tiles, splits, waves_per_row, slots;
  int narrow;                          // forward: tiles of 32 keys (see plan)
  int sink_tiles, far_chunks, far_steps, chunks, chunk_steps;   // dk and dv: see chunk_plan
  int left, right, sinks;
  float scale, scale_log2;
};

struct Sequence {
  int len, start, live;
};

__device__ __forceinline__ int clamp_length(const void* p, int is64, int b, int limit) {
  if (!p) return limit;
  const int64_t n = is64 ? reinterpret_cast<const int64_t*>(p)[b] : (int64_t)reinterpret_cast<const int*>(p)[b];
  return (int)(n < 0 ? 0 : n > limit ? limit : n);
}

__device__ __forceinline__ Sequence sequence_of(const AttentionArgs& a, int b) {
  Sequence s;
  s.len = clamp_length(a.lengths, a.lengths64, b, a.keys);
  const int rows = clamp_length(a.query_lengths, a.lengths64, b, a.rows);
  s.start = s.len > rows ? s.len - rows : 0;
  s.live = s.len < rows ? s.len : rows;
  return s;
}

// Keys that some row of the tokens [first, last] sees: [lo, hi) and the first `sinks`.
struct KeyRange {
  int lo, hi, sinks;
};

__device__ __forceinline__ KeyRange keys_of(const AttentionArgs& a, const Sequence& s, int first, int last) {
  KeyRange r;
  r.lo = max(first - a.left, 0);
  r.hi = min(last + a.right + 1, s.len);
  r.sinks = min(a.sinks, a.causal ? last + 1 : s.len);
  return r;
}

// How many of the first rows see at most `most` keys each: all of them, those of the first tokens of a causal
// sequence, or none that is known to.
__device__ __forceinline__ int rows_that_see(const AttentionArgs& a, const Sequence& s, int most) {
  if (s.len <= most || a.left + a.right + a.sinks < most) return a.rows * a.group;
  return a.causal ? max(most - s.start, 0) * a.group : 0;
}
// Rows that see no more keys than this form their output and gradients without rounding the probabilities
// and ds: the sum of few roundings does not average out, and an output's reaches all of a row's gradients
// through delta (13 tokens in bf16: dq 2.0 times as far off as its own rounding alone, 512 tokens 1.52 times;
// with exact outputs 1.4, with ds exact too 1.0 and 1.4 times).  Beyond it, second products for all keys would cost
// a quarter of a step.  dk and dv go by the extents: all rows see few keys, or none is treated so.
constexpr int kFewKeys = 128;

// The keys of a range as one list, which is walked over in tiles: place v of the list is key v for the
// sinks (v < sinks) and key v + shift for the others (v >= begin).  The two parts follow each other
// without a gap, so that a few sinks cost no tile of their own and the first tile of a window starts at
// its first key, unless a tile that holds both would span more than a buffer offset can reach.
struct KeyWalk {
  int sinks, begin, end, shift;
  __device__ __forceinline__ KeyWalk(const KeyRange& r, int64_t token_bytes, int tile) {
    if (r.sinks >= r.lo) {             // one part
      sinks = begin = shift = 0;
      end = max(r.hi, r.sinks);
    } else {
      sinks = r.sinks;
      begin = sinks % tile != 0 && (r.lo + tile) * token_bytes > 0x7fff0000 ? (sinks + tile - 1) / tile * tile : sinks;
      shift = r.lo - begin;
      end = r.hi - shift;
    }
  }
  // Bytes from the tile's first key (place v0) to place v0 + r; negative where there is none.
  __device__ __forceinline__ int offset(int v0, int r, int token_bytes) const {
    const int v = v0 + r;
    if (v < sinks) return r * token_bytes;
    return v >= begin && v < end ? (r + (v0 < begin ? shift : 0)) * token_bytes : -1;
  }
  __device__ __forceinline__ int first_key(int v0) const { return v0 < begin ? v0 : v0 + shift; }
};

// Which piece of which head a workgroup takes: the pieces of a head stay on one XCD (workgroups go to
// the 8 XCDs in turn), whose L2 then holds the head's keys and values, and four heads at a time come in
// order of rank, which the callers make the order of falling work.  Heads beyond a multiple of 8 are
// spread over all XCDs, every other round of 8 in reverse, so that none gets the heavier piece each
// time.  (Heads in plain order leave pieces of equal rank to the same XCD: causal, 32 pieces, 38 % of the
// CU time was idle.)
struct Piece {
  int rank, bh;
};
__device__ __forceinline__ Piece piece_of(int id, int pieces, int heads) {
  const int whole = heads & ~7;
  if (id < whole * pieces) {
    const int n = id >> 3, block = n / (4 * pieces);
    const int size = min(whole / 8 - block * 4, 4), at = n - block * 4 * pieces;
    const int rank = at / size;
    return {rank, (block * 4 + at - rank * size) * 8 + (id & 7)};
  }
  const int rest = heads - whole;
  id -= whole * pieces;
  if ((id & 8) && (id | 7) < rest * pieces) id ^= 7;
  return {id / rest, whole + id % rest};
}

// ---- matrix-core fragments --------------------------------------------------------------------
// A fragment holds 8 contraction elements of one row (lane % 32) per lane.  In "row" order they are
// the elements 8 h .. 8 h + 7 of a step of 16 (h = lane / 32); in "accumulator" order they are
// the elements 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3, which is how a 32 x 32 result leaves the
// matrix cores: a result whose rows are contracted next is then an operand as it stands, and only
// the other operand's reads have to follow the order (a contraction may be summed in any order).
template <typename T> struct Frag {
  typedef uint4 type;
  static __device__ __forceinline__ type zero() { return make_uint4(0u, 0u, 0u, 0u); }
  static __device__ __forceinline__ type load(const char* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ type pack(const float (&f)[8]) { return pack16<T>(f); }
  static __device__ __forceinline__ void unpack(const type& x, float (&f)[8]) { unpack16<T>(x, f); }
  // c0 += x0 y0^T and c1 += x1 y1^T
  static __device__ __forceinline__ void mma2(const type& x0, const type& y0, f32x16& c0, const type& x1, const type& y1,
                                              f32x16& c1) {
    c0 = Mfma16<T>::run(x0, y0, c0);
    c1 = Mfma16<T>::run(x1, y1, c1);
  }
  // c[n] += x(n) y^T
  template <int N, typename X> static __device__ __forceinline__ void mma_all(X&& x, const type& y, f32x16 (&c)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = Mfma16<T>::run(x(n), y, c[n]);
  }
};
struct Frag32 { float e[8]; };
template <> struct Frag<float> {
  typedef Frag32 type;
  static __device__ __forceinline__ type zero() { return type{{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}}; }
  static __device__ __forceinline__ type load(const char* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    return type{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  static __device__ __forceinline__ type pack(const float (&f)[8]) {
    return type{{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}};
  }
  static __device__ __forceinline__ void unpack(const type& x, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = x.e[j];
  }
  // eight steps of two elements each: element j of either half, in whatever order the fragments are;
  // two sums in turn, since one would wait for each step's result
  static __device__ __forceinline__ void mma2(const type& x0, const type& y0, f32x16& c0, const type& x1, const type& y1,
                                              f32x16& c1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c0 = __builtin_amdgcn_mfma_f32_32x32x2f32(x0.e[j], y0.e[j], c0, 0, 0, 0);
      c1 = __builtin_amdgcn_mfma_f32_32x32x2f32(x1.e[j], y1.e[j], c1, 0, 0, 0);
    }
  }
  template <int N, typename X> static __device__ __forceinline__ void mma_all(X&& x, const type& y, f32x16 (&c)[N]) {
    type f[N];
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = x(n);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int n = 0; n < N; ++n) c[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[n].e[j], y.e[j], c[n], 0, 0, 0);
  }
};

// What the rounding in pack(f) leaves over.
template <typename T> __device__ __forceinline__ typename Frag<T>::type low_part(const float (&f)[8]) {
  float r[8];
  Frag<T>::unpack(Frag<T>::pack(f), r);
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = f[e] - r[e];
  return Frag<T>::pack(r);
}

// Probabilities of fp16 inputs are multiplied by 2^value before they are rounded to fp16: without it
// those of a long flat row would be subnormal numbers.  In the backward pass they are at most 1, in the
// forward pass at most 2^kSlack (see there), so nothing overflows.  bf16 has fp32's exponents and needs
// no such factor.
constexpr float kSlack = 8.f;
template <typename T> struct ProbShift { static constexpr float forward = 0.f, backward = 0.f; };
template <> struct ProbShift<f16_t> { static constexpr float forward = 15.f - kSlack, backward = 15.f; };

// ds of fp16 inputs carries a factor of its own into its rounding, the same power of two for all terms of a sum (a
// row's of dq, a key's of dk), which leaves the sum in fp32: 2^kDsShift at first, lowered where a term would
// leave fp16's range, so neither small output gradients over many keys (ds is their size times a probability)
// nor large ones are lost while the sums themselves fit fp16.  As it stands, ds would be subnormal
// below 6e-5: dq of 4096 tokens was 3 to 7 times as far off as its last rounding alone with output gradients of 1e-3,
// and infinite where ds passed 65504.  With 2^11 a small term loses at most 2^-36: 2^12 of them, all
// off to the same side, make up a gradient's own smallest step.  Looking for the largest term takes 2 us of the
// 75 of a ragged batch's two kernels (6 x 1537 tokens, 12 heads on 4 of 80); with 2^15 at first, which lowers
// factors in most walks, 5 us.
// ds_factor: what brings terms of magnitude `top` > kDsLimit down to [2^12, 2^13), and its exponent.
constexpr float kDsShift = 11.f, kDsStart = 2048.f;
constexpr float kDsLimit = 32768.f;
struct DsFactor {
  float value, log2;
};
__device__ __forceinline__ DsFactor ds_factor(float top) {
  if (!(top > kDsLimit)) return {1.f, 0.f};
  const int exponent = 12 + 127 - (int)(__float_as_uint(top) >> 23);    // -116 for infinity
  return {__uint_as_float((unsigned)(exponent + 127) << 23), (float)exponent};
}
__device__ __forceinline__ float largest(const f32x16& v) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(top, fabsf(v[e])), fabsf(v[e + 1]));
  return top;
}
// 1 / x of a power of two
__device__ __forceinline__ float inverse_power(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

__device__ __forceinline__ f32x16 zero_acc() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// Value of the lane whose number differs by 32, combined with this lane's.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Row of a 32 x 32 result that register e of this lane holds.
__device__ __forceinline__ int acc_row(int e, int half) { return (e >> 2) * 8 + half * 4 + (e & 3); }

// Global -> LDS without passing through registers, as lds_dma_16, with a uniform part of the offset.
__device__ __forceinline__ void dma_16(const i32x4& rsrc, int lane_bytes, int uniform_bytes, const char* lds_dst) {
  const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(uintptr_t)lds_dst);
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(lane_bytes), "s"(rsrc),
               "s"(uniform_bytes)
               : "m0");
}

// ---- tiles in LDS -------------------------------------------------------------------------
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;

// [ROWS][dim] tile, dim padded with zeros to DT * 32 elements, rows of 64 (DT <= 2) or 128 elements.
// The 16-byte chunks of a row are permuted by an XOR with spread(row) so that both kinds of fragment
// reads touch each of the 64 banks once per pass: 16 consecutive rows at one chunk (row order), and 4
// consecutive rows at four neighbouring chunks (transposed reads).  Counted over whole passes, no cycle
// is lost to conflicts; it was a third of the forward pass's reads where only two neighbouring chunks of
// the four were apart (window of 1024 over 8192 tokens: the three kernels 1467 -> 1448 us).
template <typename T, int DT> struct Tile {
  static constexpr int kPitch = (DT <= 2 ? 64 : 128) * (int)sizeof(T);
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kSteps = 2 * DT;             // contraction steps of 16 over dim

  static __device__ __forceinline__ int spread(int row) {
    return kChunks >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  }
  // Where a lane reads: byte addresses in LDS of its first fragments of a tile.  Tiles start at multiples of
  // kPitch, so a step along dim is an XOR with a constant, and rows further down are immediate offsets:
  // two registers serve all reads of a stage.
  struct Reader {
    int rows, cols;
  };
  static __device__ __forceinline__ Reader reader(const char* stage) {
    const int lane = threadIdx.x & 63, half = lane >> 5, low = lane & 31;
    const int base = (int)(uintptr_t)(lds_char*)stage;
    Reader r;
    r.rows = base + low * kPitch + (((sizeof(T) == 2 ? half : half * 2) ^ spread(low)) << 4);
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, row = half * 4 + (i >> 2);
      r.cols = base + row * kPitch + (((((lane >> 4) & 1) * 2 + ((i & 3) >> 1)) ^ spread(row)) << 4) + (i & 1) * 8;
    } else {
      r.cols = base + half * 4 * kPitch + (((low >> 2) ^ spread(half * 4)) << 4) + (low & 3) * 4;
    }
    return r;
  }

  // Rows `row_base` + lane % 32 of the tile `tile` bytes into the stage, elements 16 step .. 16 step + 15, row order.
  static __device__ __forceinline__ typename Frag<T>::type rows_frag(const Reader& r, int tile, int row_base, int step) {
    const int off = tile + row_base * kPitch;
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(uint4, *(const lds_i32x4*)((lds_char*)(r.rows ^ (step << 5)) + off));
    } else {
      const float4 a = __builtin_bit_cast(float4, *(const lds_i32x4*)((lds_char*)(r.rows ^ (step << 6)) + off));
      const float4 b = __builtin_bit_cast(float4, *(const lds_i32x4*)((lds_char*)(r.rows ^ (step << 6) ^ 16) + off));
      return Frag32{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
  }

  // Elements (columns) 32 dt + lane % 32 as rows, tile rows `row_base` .. + 15 as contraction in
  // accumulator order.  16-bit elements are transposed by the reads themselves
  // (ds_read_b64_tr_b16: within 16 lanes, result[l][e] = source[4 e + l / 4][l % 4]).
  static __device__ __forceinline__ typename Frag<T>::type cols_frag(const Reader& r, int tile, int row_base, int dt) {
    const int off = tile + row_base * kPitch;
    if constexpr (sizeof(T) == 2) {
      const int at = r.cols ^ (dt << 6);
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)((lds_char*)at + off)));
      const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)((lds_char*)(at ^ (spread(8) << 4)) + off + 8 * kPitch)));
      return make_uint4(a.x, a.y, b.x, b.y);
    } else {
      Frag32 f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = (j < 4 ? 0 : 8) + (j & 3);
        f.e[j] = *(const lds_float*)((lds_char*)(r.cols ^ (dt << 7) ^ (spread(row) << 4)) + off + row * kPitch);
      }
      return f;
    }
  }

  // ---- asynchronous copies of ROWS rows into a tile, shared among NW waves ----
  // A wave moves kLoadRows rows with one load and NW * kLoadRows with all waves' loads (a round).  The
  // chunk a lane moves is the same in every round but for the part of spread() that the round sets.
  static constexpr int kLoadRows = 1024 / kPitch;
  template <int NW> static __device__ __forceinline__ int lane_row() {
    return ((int)threadIdx.x >> 6) * kLoadRows + ((int)threadIdx.x & 63) / kChunks;
  }
  template <int NW> static __device__ __forceinline__ int lane_byte(int round) {
    const int chunk = ((int)threadIdx.x & 63) % kChunks;
    return (chunk ^ spread(lane_row<NW>()) ^ spread(round * NW * kLoadRows)) << 4;
  }
  // Byte offset of a lane's part of a row that lies `row_bytes` behind the tile's first: kOobOffset where the
  // row has no such part.
  template <int NW> static __device__ __forceinline__ int lane_offset(int row_bytes, int dim_bytes, int round) {
    const int byte = lane_byte<NW>(round);
    return byte < dim_bytes ? row_bytes + byte : kOobOffset;
  }

  // Every row exists, and rounds lie `round_bytes` apart: lane offsets do not change from tile to tile.
  template <int ROWS, int NW>
  static __device__ __forceinline__ void fetch_all(const i32x4& rsrc, const int (&offset)[2], int round_bytes, char* tile) {
    constexpr int kRounds = ROWS / (NW * kLoadRows);
    static_assert(kRounds * NW * kLoadRows == ROWS, "every wave issues the same number of loads");
    char* dst = tile + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int n = 0; n < kRounds; ++n)
      dma_16(rsrc, offset[spread(n * NW * kLoadRows) != 0], n * round_bytes, dst + n * NW * 1024);
  }

  // offset(row) is the row's byte offset from the tile's first, negative for a row that is to be zeros.
  template <int ROWS, int NW, typename Offset>
  static __device__ __forceinline__ void fetch(const i32x4& rsrc, int dim_bytes, char* tile, Offset&& offset) {
    constexpr int kRounds = ROWS / (NW * kLoadRows);
    char* dst = tile + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * 1024;
    int row = lane_row<NW>();
    asm volatile("" : "+v"(row));      // nothing of this rare path is to be kept in registers between tiles
#pragma unroll
    for (int n = 0; n < kRounds; ++n) {
      const int off = offset(row + n * NW * kLoadRows);
      dma_16(rsrc, off >= 0 ? lane_offset<NW>(off, dim_bytes, n) : kOobOffset, 0, dst + n * NW * 1024);
    }
  }
};

// A wave's accumulators through LDS, one word per lane and step: `room` bytes serve a wave.
template <int N> struct Exchange {
  static constexpr int kBytes = N * 256;
  template <int M> static __device__ __forceinline__ void put(char* room, int first, const f32x16 (&v)[M]) {
    float* p = reinterpret_cast<float*>(room) + (threadIdx.x & 63) + first * 64;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e) p[(m * 16 + e) * 64] = v[m][e];
  }
  static __device__ __forceinline__ float get(const char* room, int at) {
    return reinterpret_cast<const float*>(room)[at * 64 + (threadIdx.x & 63)];
  }
};

// Resource of everything from `base` on; rows that must not be read get kOobOffset.
__device__ __forceinline__ i32x4 open_rsrc(const char* base) {
  i32x4 r = make_buffer_rsrc(base, 0x7fffffff);
  r.x = __builtin_amdgcn_readfirstlane(r.x);
  r.y = __builtin_amdgcn_readfirstlane(r.y);
  return r;
}

// ---- host side ----------------------------------------------------------------------------
constexpr int kRowAlign = 64;          // rows of lse and delta are padded to whole tiles

inline int workgroups_per_cu(int dtype, int dim) { return dtype == AT_DTYPE_F32 && dim > 64 ? 1 : 2; }

// Waves that share 32 rows and halve each tile of keys (kernels that own rows): two where workgroups of
// whole rows leave some of the GPU's `slots` for workgroups empty.  Sharing reads keys and values twice as
// often, empty slots cost more (a chunk of 1024 over 16384 keys, bf16: 256 workgroups on 512 slots 107 us,
// split and joined 92 us, shared 93 us without the join's workspace; fp32 patches: dq 88 -> 52 us; fp32,
// causal, 4486 tokens, 282 workgroups: dq 98 -> 57 us; with all slots taken, a block of 512 tokens: 27 -> 30 us).
inline int waves_per_row(int64_t rows, int64_t heads, int64_t slots) { return cdiv64(rows, 128) * heads < slots ? 2 : 1; }

inline bool grid_fits(int64_t workgroups) { return workgroups < ((int64_t)1 << 24); }   // 256 threads each, 32-bit grid

// Checks the shape and fills the arguments that do not depend on the pointers.
inline int attention_args(const at_attention_t* s, AttentionArgs& a) {
  if (!s) return AT_ERR_NULL;
  if (!dtype_valid(s->dtype)) return AT_ERR_DTYPE;
  const int64_t limit = (int64_t)1 << 29;
  if (s->batch < 0 || s->batch > 65535 || s->kv_heads <= 0 || s->kv_heads > 65535 || s->heads <= 0 || s->heads > 65535 ||
      s->heads % s->kv_heads != 0 || s->rows < 0 || s->keys < s->rows || s->keys > limit || s->dim <= 0 || s->dim > 128 ||
      s->window < 0 || s->sinks < 0)
    return AT_ERR_DIM;
  if (!(s->scale > 0.f) || s->scale > 1e38f) return AT_ERR_DIM;
  if (s->dim % 8 != 0) return AT_ERR_ALIGN;
  a = AttentionArgs{};
  a.batch = (int)s->batch;
  a.kv_heads = (int)s->kv_heads;
  a.group = (int)(s->heads / s->kv_heads);
  a.rows = (int)s->rows;
  a.keys = (int)s->keys;
  a.dim = (int)s->dim;
  if (s->rows * a.group > limit) return AT_ERR_DIM;
  a.row_pitch = (int)(cdiv64(s->rows * a.group, kRowAlign) * kRowAlign);
  const int64_t reach = s->window > 0 && s->window - 1 < s->keys ? s->window - 1 : s->keys;
  a.left = (int)reach;
  a.right = s->causal ? 0 : (int)reach;
  a.sinks = (int)(s->sinks < s->keys ? s->sinks : s->keys);
  a.causal = s->causal != 0;
  a.slots = workgroups_per_cu(s->dtype, a.dim) * device_cu_count();
  a.scale = s->scale;
  a.scale_log2 = s->scale * kLog2E;
  a.lengths64 = s->lengths_int64;
  const int size = dtype_size(s->dtype);
  Strided* const views[8] = {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv};
  for (int n = 0; n < 8; ++n) {
    const int64_t* st = s->strides[n];
    for (int j = 0; j < 3; ++j) {
      if (st[j] < 0 || st[j] > ((int64_t)1 << 56)) return AT_ERR_DIM;
      if (st[j] * size % 16 != 0) return AT_ERR_ALIGN;
    }
    *views[n] = Strided{nullptr, st[0] * size, st[1] * size, st[2] * size};
    // a tile is read with 32-bit offsets from its first token
    const bool heads_in_tile = n == 0 || n == 4;
    const double span = 160.0 * (double)(st[2] * size) + (heads_in_tile ? (double)(a.group - 1) * (double)(st[1] * size) : 0.0);
    if (n < 3 || n == 4) { if (span >= 2147483000.0) return AT_ERR_DIM; }
  }
  return AT_OK;
}

}  // namespace at_hip
