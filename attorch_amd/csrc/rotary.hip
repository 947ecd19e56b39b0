// Rotary positions with one or several axes: pair n of each head's features is turned by the angle
//   a = positions[axis of n] * inv_freq[n]:   (x, y) -> (x cos a - y sin a, x sin a + y cos a).
// The gradient is the same map with -a, so one kernel serves both directions.
//
// Bound by memory: every feature is read and written once.  A workgroup takes a few tokens, forms the
// cosines and sines of their angles and the tokens' addresses once in LDS (all heads of a token share
// them) and then streams the heads of q and k.  A lane keeps its place in a head and goes from head to
// head, two at a time, so that it has four vectors in flight.  The angles are formed in 64 bits and
// reduced by whole turns there: at position 2^20 an fp32 product would already be off by 0.06 radians.
#include "at_common.h"

namespace at_hip {
namespace {

constexpr int kMaxPairs = 512;
constexpr int kTable = 1024;           // cosines and sines in LDS
constexpr int kMaxTokens = 8;          // of a workgroup

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
};

__device__ __forceinline__ double position_of(const RotaryArgs& a, int axis, int64_t b, int t) {
  if (!a.positions) return (double)t;
  const int64_t at = axis * a.position_strides[0] + b * a.position_strides[1] + t * a.position_strides[2];
  if (a.position_type == 0) return (double)reinterpret_cast<const int*>(a.positions)[at];
  if (a.position_type == 1) return (double)reinterpret_cast<const int64_t*>(a.positions)[at];
  return (double)reinterpret_cast<const float*>(a.positions)[at];
}

// What a lane turns or copies at a time: VEC features (1: any size and alignment) of either half of the
// pairs, or of adjacent pairs, or of the rest.
template <typename T, bool ADJACENT, int VEC> struct Item {
  static constexpr int kWidth = VEC > 1 || !ADJACENT ? VEC : 2;    // features an adjacent item covers
  static constexpr bool kTwo = !ADJACENT;                          // two places in a head
  float u[kWidth], w[kTwo ? VEC : 1];

  static __device__ __forceinline__ void read(const T* p, float (&v)[kWidth]) {
    if constexpr (VEC > 1 || kWidth == 1) {
      load_f32<T, kWidth>(p, v);
    } else {
      v[0] = to_f32(p[0]);
      v[1] = to_f32(p[1]);
    }
  }
  static __device__ __forceinline__ void write(T* p, const float (&v)[kWidth]) {
    if constexpr (VEC > 1 || kWidth == 1) {
      store_f32<T, kWidth>(p, v);
    } else {
      p[0] = from_f32<T>(v[0]);
      p[1] = from_f32<T>(v[1]);
    }
  }
  __device__ __forceinline__ void load(const T* head, int d, int pairs) {
    read(head + d, u);
    if constexpr (kTwo) load_f32<T, VEC>(head + d + pairs, w);
  }
  __device__ __forceinline__ void turn(const float* cs, const float* sn, int d) {
    if constexpr (kTwo) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float c = cs[d + j], s = sn[d + j], x = u[j], y = w[j];
        u[j] = x * c - y * s;
        w[j] = x * s + y * c;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kWidth; j += 2) {
        const float c = cs[(d + j) >> 1], s = sn[(d + j) >> 1], x = u[j], y = u[j + 1];
        u[j] = x * c - y * s;
        u[j + 1] = x * s + y * c;
      }
    }
  }
  __device__ __forceinline__ void store(T* head, int d, int pairs) const {
    write(head + d, u);
    if constexpr (kTwo) store_f32<T, VEC>(head + d + pairs, w);
  }
};

template <typename T, bool ADJACENT, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  typedef Item<T, ADJACENT, VEC> I;
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

  // places of a head: items of pairs, then vectors of the features that are only copied
  const int turned = ADJACENT ? 2 * a.pairs / I::kWidth : a.pairs / VEC;
  const int places = turned + (a.dim - 2 * a.pairs) / VEC;
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
  for (int place = (int)threadIdx.x - mine * across; place < places; place += across) {
    if (place < turned) {
      const int d = place * I::kWidth;
      int n = mine;
      for (; n + step < heads; n += 2 * step) {
        const T *x0, *x1;
        T *y0, *y1;
        int t0, t1;
        find(n, x0, y0, t0);
        find(n + step, x1, y1, t1);
        I i0, i1;
        i0.load(x0, d, a.pairs);
        i1.load(x1, d, a.pairs);
        i0.turn(table_cos + t0 * a.pairs, table_sin + t0 * a.pairs, d);
        i0.store(y0, d, a.pairs);
        i1.turn(table_cos + t1 * a.pairs, table_sin + t1 * a.pairs, d);
        i1.store(y1, d, a.pairs);
      }
      if (n < heads) {
        const T* x;
        T* y;
        int t;
        find(n, x, y, t);
        I i;
        i.load(x, d, a.pairs);
        i.turn(table_cos + t * a.pairs, table_sin + t * a.pairs, d);
        i.store(y, d, a.pairs);
      }
    } else {
      const int d = 2 * a.pairs + (place - turned) * VEC;
      for (int n = mine; n < heads; n += step) {
        const T* x;
        T* y;
        int t;
        find(n, x, y, t);
        float v[VEC];
        load_f32<T, VEC>(x + d, v);
        store_f32<T, VEC>(y + d, v);
      }
    }
  }
}

template <typename T, int VEC>
int launch(const RotaryArgs& a, bool adjacent, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv64(a.tokens, a.group)), block(256);
  if (adjacent) hipLaunchKernelGGL((rotary_kernel<T, true, VEC>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, false, VEC>), grid, block, 0, stream, a);
  return launch_status();
}

template <typename T>
int launch_width(const RotaryArgs& a, bool adjacent, int width, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (width == 8) return launch<T, 8>(a, adjacent, stream);
  }
  if (width >= 4) return launch<T, 4>(a, adjacent, stream);
  if (width >= 2) return launch<T, 2>(a, adjacent, stream);
  return launch<T, 1>(a, adjacent, stream);
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
  // features of an access: the largest power of two that the pairs (both halves of them, or adjacent
  // ones), the head, the strides and the addresses are multiples of, up to 16 bytes
  int64_t common = (s->adjacent ? 2 * s->pairs : s->pairs) | s->dim | 16 / size;
  int64_t bytes = 16;
  for (int n = 0; n < 2; ++n) {
    if ((n == 0 ? s->q_heads : s->k_heads) == 0) continue;
    bytes |= (int64_t)(uintptr_t)a.in[n] | (int64_t)(uintptr_t)a.out[n];
    for (int j = 0; j < 3; ++j) {
      a.in_stride[n][j] = s->strides[n][j] * size;
      a.out_stride[n][j] = s->strides[2 + n][j] * size;
      bytes |= a.in_stride[n][j] | a.out_stride[n][j];
    }
  }
  common |= (bytes & -bytes) / size;
  const int width = (int)(common & -common);
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
  // tokens of a workgroup: as many as fill its lanes with angles, as long as every CU keeps several workgroups
  int group = a.pairs > 0 ? 256 / a.pairs : 4;
  if (group > kMaxTokens) group = kMaxTokens;
  while (group > 1 && a.tokens / group < 4 * (int64_t)device_cu_count()) group /= 2;
  a.group = group < 1 ? 1 : group;
  if (cdiv64(a.tokens, a.group) >= ((int64_t)1 << 24)) return AT_ERR_DIM;
  if (s->dtype == AT_DTYPE_F32) return launch_width<float>(a, s->adjacent != 0, width, (hipStream_t)stream);
  if (s->dtype == AT_DTYPE_F16) return launch_width<f16_t>(a, s->adjacent != 0, width, (hipStream_t)stream);
  return launch_width<bf16_t>(a, s->adjacent != 0, width, (hipStream_t)stream);
}

}  // extern "C"
