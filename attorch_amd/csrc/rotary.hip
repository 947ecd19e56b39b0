// Rotary positions with one or several axes: pair n of each head's features is turned by the angle
//   a = positions[axis of n] * inv_freq[n]:   (x, y) -> (x cos a - y sin a, x sin a + y cos a).
// The gradient is the same map with -a, so one kernel serves both directions.
//
// Bound by memory: every feature is read and written once.  A workgroup takes a few tokens, forms the
// cosines and sines of their angles and the tokens' addresses once in LDS (all heads of a token share
// them) and then streams the heads of q and k.  A lane keeps its place in a head and goes from head to
// head, two at a time, so that it has four vectors in flight; lanes that only copy run along with those
// that turn, and select instead of branching (a branch holds the loads of the tables back until those
// of the features are there: 51 instead of 31 us for 8 x 4096 tokens of 24 heads of 64 features).  The
// angles are formed in 64 bits and reduced by whole turns there: at position 2^20 an fp32 product would
// already be off by 0.06 radians; the rest of the turn, its cosine and sine and the products are fp32.  Results are
// rounded once more, to the type of the inputs.
//
// 8 x 4096 tokens, 24 heads of 128 features, bf16: 75 us (5.4 TB/s); fp32 147 us (5.5 TB/s); a quarter of
// the features turned 79 us; 5 or 37 pairs of 80 features, whose halves start anywhere, 40 us (6.3 TB/s, in
// part from the last level cache).  One token of 128 sequences: 8 us, the latency of the launch, of the
// angles' and then of the features' loads.
#include <algorithm>
#include <type_traits>

#include "at_common.h"

namespace at_hip {
namespace {

constexpr int kMaxPairs = 512;
constexpr int kTable = 1024;           // cosines and sines in LDS
constexpr int kMaxTokens = 8;          // of a workgroup

template <int W> using Width = std::integral_constant<int, W>;

struct RotaryArgs {
  const char* in[2];                   // q, k
  char* out[2];
  int64_t in_stride[2][3], out_stride[2][3];   // batch, head, token; bytes
  const void* positions;
  const double* inv_freq;
  const int* pair_axis;
  int64_t position_strides[3];
  int64_t tokens;                      // batch * rows
  int rows, heads, q_heads, dim, pairs, axes, position_type, inverse, group;
  int turn_span, turn_width, copy_span, copy_width;   // see cut()
};

__device__ __forceinline__ double position_of(const RotaryArgs& a, int axis, int64_t b, int t) {
  if (!a.positions) return (double)t;
  const int64_t at = axis * a.position_strides[0] + b * a.position_strides[1] + t * a.position_strides[2];
  if (a.position_type == 0) return (double)reinterpret_cast<const int*>(a.positions)[at];
  if (a.position_type == 1) return (double)reinterpret_cast<const int64_t*>(a.positions)[at];
  return (double)reinterpret_cast<const float*>(a.positions)[at];
}

// What a lane takes of a head at a time: W features in two places, either half of pairs or features that
// are only copied; with adjacent pairs in one place.  Lanes that turn and lanes that copy go together.
// Accesses assume no more than an element's alignment: the hardware takes a vector from any address at
// full speed, so odd sizes and strides do not make accesses narrow.
template <typename T, bool ADJACENT, int W> struct Item {
  T u[W], w[ADJACENT ? 1 : W];

  __device__ __forceinline__ void load(const T* head, int d0, int d1) {
    __builtin_memcpy(u, head + d0, W * sizeof(T));
    if constexpr (!ADJACENT) __builtin_memcpy(w, head + d1, W * sizeof(T));
  }
  static __device__ __forceinline__ void turn(T& p, T& q, float c, float s, bool turns) {
    const float x = to_f32(p), y = to_f32(q);
    p = turns ? from_f32<T>(__builtin_fmaf(-y, s, x * c)) : p;     // one order of roundings in all lanes
    q = turns ? from_f32<T>(__builtin_fmaf(y, c, x * s)) : q;
  }
  __device__ __forceinline__ void turn(const float* cs, const float* sn, bool turns) {
    if constexpr (!ADJACENT) {
#pragma unroll
      for (int j = 0; j < W; ++j) turn(u[j], w[j], cs[j], sn[j], turns);
    } else if constexpr (W > 1) {          // single features are only copied
#pragma unroll
      for (int j = 0; j < W; j += 2) turn(u[j], u[j + 1], cs[j >> 1], sn[j >> 1], turns);
    }
  }
  __device__ __forceinline__ void store(T* head, int d0, int d1) const {
    __builtin_memcpy(head + d0, u, W * sizeof(T));
    if constexpr (!ADJACENT) __builtin_memcpy(head + d1, w, W * sizeof(T));
  }
};

__host__ __device__ __forceinline__ int items(int span, int width) { return (span + width - 1) / width; }

template <typename T, bool ADJACENT>
__global__ __launch_bounds__(256, 6) void rotary_kernel(RotaryArgs a) {
  __shared__ float table_cos[kTable], table_sin[kTable];
  __shared__ int64_t base[kMaxTokens][4];      // token's offsets in q, k, q_out, k_out
  const int64_t first = (int64_t)blockIdx.x * a.group;
  const int count = (int)(a.tokens - first < a.group ? a.tokens - first : a.group);

  if ((int)threadIdx.x < count) {
    const int64_t b = (first + threadIdx.x) / a.rows, t = first + threadIdx.x - b * a.rows;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      base[threadIdx.x][n] = b * a.in_stride[n][0] + t * a.in_stride[n][2];
      base[threadIdx.x][2 + n] = b * a.out_stride[n][0] + t * a.out_stride[n][2];
    }
  }
  for (int n = threadIdx.x; n < count * a.pairs; n += 256) {
    const int local = n / a.pairs, pair = n - local * a.pairs;
    const int64_t b = (first + local) / a.rows;
    const int t = (int)(first + local - b * a.rows);
    const int axis = a.pair_axis ? min(max(a.pair_axis[pair], 0), a.axes - 1) : 0;
    const double turns = position_of(a, axis, b, t) * (a.inv_freq[pair] * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    table_cos[n] = c;
    table_sin[n] = a.inverse ? -s : s;
  }
  __syncthreads();

  const int turned = items(a.turn_span, a.turn_width), places = turned + items(a.copy_span, a.copy_width);
  const int across = places < 256 ? places : 256, step = 256 / across;
  const int mine = (int)threadIdx.x / across;
  if (mine >= step) return;
  const int heads = count * a.heads;           // of all tokens
  const float per_heads = 1.f / (float)a.heads;
  auto find = [&](int n, const T*& x, T*& y, int& local) {
    local = (int)(((float)n + 0.5f) * per_heads);   // n < 2^19: off by far less than the 0.5 / heads that would matter
    int head = n - local * a.heads;
    const int which = head >= a.q_heads;
    head -= which ? a.q_heads : 0;
    x = reinterpret_cast<const T*>(a.in[which] + base[local][which] + head * a.in_stride[which][1]);
    y = reinterpret_cast<T*>(a.out[which] + base[local][2 + which] + head * a.out_stride[which][1]);
  };
  auto go = [&](auto width, bool turns, int d0, int d1) {
    typedef Item<T, ADJACENT, decltype(width)::value> I;
    const int angle = turns ? (ADJACENT ? d0 / 2 : d0) : 0;
    const float *cs = table_cos + angle, *sn = table_sin + angle;
    int n = mine;
    for (; n + step < heads; n += 2 * step) {
      const T *x0, *x1;
      T *y0, *y1;
      int t0, t1;
      find(n, x0, y0, t0);
      find(n + step, x1, y1, t1);
      I i0, i1;
      i0.load(x0, d0, d1);
      i1.load(x1, d0, d1);
      i0.turn(cs + t0 * a.pairs, sn + t0 * a.pairs, turns);
      i0.store(y0, d0, d1);
      i1.turn(cs + t1 * a.pairs, sn + t1 * a.pairs, turns);
      i1.store(y1, d0, d1);
    }
    if (n < heads) {
      const T* x;
      T* y;
      int t;
      find(n, x, y, t);
      I i;
      i.load(x, d0, d1);
      i.turn(cs + t * a.pairs, sn + t * a.pairs, turns);
      i.store(y, d0, d1);
    }
  };
  for (int place = (int)threadIdx.x - mine * across; place < places; place += across) {
    const bool turns = place < turned;
    const int width = turns ? a.turn_width : a.copy_width;
    const int at = turns ? min(place * width, a.turn_span - width) : min((place - turned) * width, a.copy_span - width);
    const int d0 = turns ? at : 2 * a.pairs + at, d1 = turns ? at + a.pairs : a.dim - a.copy_span + at;
    if (width == 16 / (int)sizeof(T)) go(Width<16 / (int)sizeof(T)>(), turns, d0, d1);
    else if (sizeof(T) == 2 && width == 4) go(Width<4>(), turns, d0, d1);
    else if (width == 2) go(Width<2>(), turns, d0, d1);
    else if (!ADJACENT || !turns) go(Width<1>(), turns, d0, d1);
  }
}

template <typename T>
int launch(const RotaryArgs& a, bool adjacent, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv64(a.tokens, a.group)), block(256);
  if (adjacent) hipLaunchKernelGGL((rotary_kernel<T, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, false>), grid, block, 0, stream, a);
  return launch_status();
}

// Cuts a head into items.  Those of pairs cover turn_span features from 0 (the first half of the pairs: an
// item's second place lies `pairs` behind; or all adjacent ones), those of the rest copy_span features from
// 2 * pairs (second places end with the head).  The last item of either ends with the span, so it may cover
// features that others cover too: all write the same.  Only where pairs are turned in place does each
// belong to one item.  Lanes with items of two widths take turns, so both get the smaller one where that
// makes fewer than twice the items (5 pairs and 70 more features: 11 items of 4 instead of 2 of 4 and 5
// of 8, 68 -> 40 us for 8 x 4096 tokens of 24 heads).
void cut(RotaryArgs& a, int most, bool adjacent, bool in_place) {
  const int copied = a.dim - 2 * a.pairs;
  a.turn_span = adjacent ? 2 * a.pairs : a.pairs;
  a.turn_width = a.copy_width = most;
  while (a.turn_width > 1 && (a.turn_width > a.turn_span || (in_place && a.turn_span % a.turn_width != 0)))
    a.turn_width /= 2;
  while (a.copy_width > 1 && a.copy_width > copied) a.copy_width /= 2;
  auto span = [&](int width) { return adjacent || copied == 0 ? copied : std::max((copied + 1) / 2, width); };
  a.copy_span = span(a.copy_width);
  const int least = std::min(a.turn_width, a.copy_width);
  if (a.turn_span == 0 || copied == 0 || (adjacent && least < 2)) return;
  if (items(a.turn_span, least) + items(span(least), least) <
      2 * (items(a.turn_span, a.turn_width) + items(a.copy_span, a.copy_width))) {
    a.turn_width = a.copy_width = least;
    a.copy_span = span(least);
  }
}

}  // namespace
}  // namespace at_hip

using namespace at_hip;

extern "C" {

int at_rotary(const at_rotary_t* s, const void* q, const void* k, void* q_out, void* k_out, const void* positions,
              const double* inv_freq, const int* pair_axis, at_stream_t stream) {
  if (!s) return AT_ERR_NULL;
  if (!dtype_valid(s->dtype)) return AT_ERR_DTYPE;
  const int64_t limit = (int64_t)1 << 30;
  if (s->batch < 0 || s->rows < 0 || s->q_heads < 0 || s->k_heads < 0 || s->dim <= 0 || s->pairs < 0 || s->axes <= 0 ||
      s->pairs > kMaxPairs || 2 * s->pairs > s->dim || s->rows > limit || s->batch > limit ||
      s->position_type < 0 || s->position_type > 2)
    return AT_ERR_DIM;
  const int64_t heads = s->q_heads + s->k_heads;
  if (heads > 65535 || s->dim > 65535 || heads * s->dim > limit) return AT_ERR_DIM;
  if (s->batch == 0 || s->rows == 0 || heads == 0) return AT_OK;
  if ((s->q_heads > 0 && (!q || !q_out)) || (s->k_heads > 0 && (!k || !k_out)) || (s->pairs > 0 && !inv_freq) ||
      (s->axes > 1 && (!positions || (s->pairs > 0 && !pair_axis))))
    return AT_ERR_NULL;
  const int size = dtype_size(s->dtype);
  RotaryArgs a = {};
  a.in[0] = (const char*)q; a.in[1] = (const char*)k;
  a.out[0] = (char*)q_out; a.out[1] = (char*)k_out;
  for (int n = 0; n < 2; ++n) {
    for (int j = 0; j < 3; ++j) {
      a.in_stride[n][j] = s->strides[n][j] * size;
      a.out_stride[n][j] = s->strides[2 + n][j] * size;
    }
  }
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.pair_axis = pair_axis;
  for (int j = 0; j < 3; ++j) a.position_strides[j] = s->position_strides[j];
  a.tokens = s->batch * s->rows;
  a.rows = (int)s->rows;
  a.heads = (int)heads;
  a.q_heads = (int)s->q_heads;
  a.dim = (int)s->dim;
  a.pairs = (int)s->pairs;
  a.axes = (int)s->axes;
  a.position_type = s->position_type;
  a.inverse = s->inverse != 0;
  cut(a, 16 / size, s->adjacent != 0, (q && q == q_out) || (k && k == k_out));
  // tokens of a workgroup: as many as fill its lanes with angles, as long as every CU keeps several workgroups
  int group = a.pairs > 0 ? 256 / a.pairs : 4;
  if (group > kMaxTokens) group = kMaxTokens;
  while (group > 1 && a.tokens / group < 4 * (int64_t)device_cu_count()) group /= 2;
  a.group = group < 1 ? 1 : group;
  if (cdiv64(a.tokens, a.group) >= ((int64_t)1 << 24)) return AT_ERR_DIM;
  if (s->dtype == AT_DTYPE_F32) return launch<float>(a, s->adjacent != 0, (hipStream_t)stream);
  if (s->dtype == AT_DTYPE_F16) return launch<f16_t>(a, s->adjacent != 0, (hipStream_t)stream);
  return launch<bf16_t>(a, s->adjacent != 0, (hipStream_t)stream);
}

}  // extern "C"
