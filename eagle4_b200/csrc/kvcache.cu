// The paged KV cache's write side in 8 or 16 bits, and its read-back: the attention projection's post-processing with
// multi-axis rotary positions, quantisation of given K and V rows, dequantisation, and the accepted rows' moves.
//
// All four are bound by HBM: per element they read or write 1 to 4 bytes and compute about ten operations, so what counts
// besides wide accesses is to spend few instructions per element. A cache row (one token's one kv head) is handled by
// a group of up to 16 lanes of one warp, two pieces of eight elements a lane (the second piece half a row further, so
// that every access of the group is one run of 16-byte vectors): its RMS and largest magnitude are at most four
// butterfly shuffles, and what is done once per row (scale, reciprocal, address) is shared by 16 elements. Sums, norms,
// rotations and scales are fp32; the only roundings below 32 bits are the stored codes or bf16 rows. A row's result does not depend on how many rows share the launch.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "quant.cuh"

namespace e4 {

torch::Tensor gemm_error_word(torch::Device dev);

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxAxes = 4;

constexpr int kMaxLanes = 16;  // lanes of a row: two pieces of eight elements each, D <= 256

// Lanes that hold one row of D elements, as a power of two.
inline int row_lanes(int D) {
  int n = 1;
  while (n * 16 < D) n *= 2;
  return n;
}

E4_DEV uint32_t group_max(uint32_t v, int lanes) {
#pragma unroll
  for (int o = kMaxLanes / 2; o > 0; o >>= 1)
    if (o < lanes) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
E4_DEV float group_sum(float v, int lanes) {
#pragma unroll
  for (int o = kMaxLanes / 2; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

E4_DEV void unpack8(const uint4& raw, float* x, const __nv_bfloat16*) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(p[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}
E4_DEV void unpack8(const uint4& raw, float* x, const __half*) {
  const __half2* p = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(p[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}
E4_DEV uint4 pack8(const float* x, const __nv_bfloat16*) {
  uint4 r;
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
  return r;
}
E4_DEV uint4 pack8(const float* x, const __half*) {
  uint4 r;
  __half2* p = reinterpret_cast<__half2*>(&r);
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
  return r;
}

// Eight elements as they lie in memory: two or four 16-byte vectors' worth, loaded whole when ``vec`` (the pointer and
// every stride keep 16-byte alignment), else one by one.
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];
  E4_DEV void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  E4_DEV void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w)[i] = p[i];
    }
  }
  E4_DEV void get(float* x) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
      unpack8(make_uint4(w[0], w[1], w[2], w[3]), x, (const T*)nullptr);
    }
  }
  // The largest |x|'s bit pattern as fp32 (16-bit types: two maxima an instruction on the raw patterns, whose order is
  // the magnitudes')
  E4_DEV uint32_t amax() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      const uint32_t k = 0x7fff7fffu;
      uint32_t m = __vimax3_u16x2(w[0] & k, w[1] & k, w[2] & k);
      m = __vimax3_u16x2(m, w[3] & k, m);
      m = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
      else return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
    }
  }
};

E4_DEV uint32_t amax8(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

// Writes this lane's pieces (element i0 and, ``second`` elements on, the other one; ``on``: whether each exists) of the
// cache row (slot, h), given the row's scale: codes and, in the group's first lane, the scale; or bf16 elements.
template <int FMT>
E4_DEV void write_row(const float (*x)[8], int i0, int second, const bool* on, float s, void* data, float* scale,
                      int64_t slot, int64_t slots, int h, int Hk, int D) {
  const size_t at = (size_t(slot) * Hk + h) * D + i0;
  if constexpr (FMT == kFmtBf16) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (on[j])
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(data) + at + j * second) =
            pack8(x[j], (const __nv_bfloat16*)nullptr);
  } else {
    const float inv = inv_of(s);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (on[j])
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(data) + at + j * second) =
            make_uint2(encode4<FMT>(x[j], inv, s == s), encode4<FMT>(x[j] + 4, inv, s == s));
    if (on[0] && i0 == 0) scale[size_t(h) * slots + slot] = s;
  }
}

struct PrepareArgs {
  const __nv_bfloat16* qkv;
  const int64_t* pos;   // [axes, T]
  const int64_t* slot;  // [T]
  const __nv_bfloat16 *qn, *kn;
  const double* inv;    // [rot / 2] turns per position
  void *k, *v;
  float *ks, *vs;
  __nv_bfloat16* q;
  int* err;
  int64_t slots, ldq, pos_ld;
  int Hq, Hk, D, rot, lanes, koff, axes, sec[kMaxAxes];
  int interleaved, norm_offset;
  float eps, inv_d;
};

// The axis whose position turns frequency j: consecutive sections, or axis a at a, a + axes, ... (its section's count
// of them), axis 0 elsewhere.
E4_DEV int axis_of(const PrepareArgs& p, int j) {
  if (p.axes == 1) return 0;
  if (p.interleaved) {
    const int a = j % p.axes;
    return a > 0 && j < p.axes * p.sec[a] ? a : 0;
  }
  int a = 0, end = p.sec[0];
  while (a + 1 < p.axes && j >= end) end += p.sec[++a];
  return a;
}

// One block per row (grid.y more of them share a row's heads): the angles' cos and sin once per block, then every lane
// group takes head rows [q heads | k heads | v heads] in turn, the next one's load in flight while it works. The angle
// is reduced in whole turns in fp64 (position * turns per position, minus its nearest integer), so a position of any
// size keeps fp32 accuracy and no table bounds the positions. Bound by instructions and the chain before a block's
// first store, not yet by HBM: 8192 rows of 24 + 4 + 4 heads x 256 with norms into int8 take 74 us (3.4 TB/s, half of
// the copy rate) at four blocks an SM, 111 us at two.
template <int FMT>
__global__ void __launch_bounds__(kThreads, 4) prepare_axes_kernel(const PrepareArgs p) {
  pdl_wait();
  pdl_trigger();
  __shared__ __align__(16) float cs[128], sn[128];
  __shared__ __align__(16) float buf[kWarps][32 * 16];
  const int64_t r = blockIdx.x;
  const int half = p.rot / 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gpw = 32 / p.lanes, sub = lane / p.lanes, i0 = (lane % p.lanes) * 8, second = p.lanes * 8;
  const int total = p.Hq + 2 * p.Hk, step = gridDim.y * kWarps * gpw;
  const __nv_bfloat16* row = p.qkv + r * p.ldq + i0;
  auto fetch = [&](int hh, uint4* raw) {
    const __nv_bfloat16* src = row + (hh < p.Hq ? hh * p.D : p.koff + (hh - p.Hq) * p.D);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      raw[j] = hh < total && i0 + j * second < p.D ? *reinterpret_cast<const uint4*>(src + j * second)
                                                   : make_uint4(0, 0, 0, 0);
  };
  int base = (blockIdx.y * kWarps + warp) * gpw;
  uint4 next[2];
  fetch(base + sub, next);
  for (int j = threadIdx.x; j < half; j += kThreads) {
    double t = double(p.pos[axis_of(p, j) * p.pos_ld + r]) * p.inv[j];
    t -= rint(t);
    sincospif(float(2.0 * t), &sn[j], &cs[j]);
  }
  const int64_t slot = p.slot[r];
  const bool keep = slot >= 0 && slot < p.slots;
  if (slot >= p.slots && threadIdx.x == 0 && blockIdx.y == 0) record_error(p.err, kErrBadIndex);
  __syncthreads();
  for (; base < total; base += step) {
    const int hh = base + sub;
    float x[2][8];
    unpack8(next[0], x[0], (const __nv_bfloat16*)nullptr);
    unpack8(next[1], x[1], (const __nv_bfloat16*)nullptr);
    fetch(hh + step, next);
    const bool isq = hh < p.Hq, isk = !isq && hh < p.Hq + p.Hk;
    const bool in[2] = {hh < total && i0 < p.D, hh < total && i0 + second < p.D};
    if (base < p.Hq + p.Hk) {  // some head of the warp is q or k
      const __nv_bfloat16* nw = isq ? p.qn : isk ? p.kn : nullptr;
      if (p.qn || p.kn) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i / 8][i % 8], x[i / 8][i % 8], ss);
        ss = group_sum(ss, p.lanes);
        if (nw) {
          const float rs = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (!in[j]) continue;
            float w[8];
            unpack8(*reinterpret_cast<const uint4*>(nw + i0 + j * second), w, nw);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float y = x[j][i] * rs;
              x[j][i] = fmaf(y, w[i], p.norm_offset ? y : 0.f);
            }
          }
        }
      }
      // pairs (i, i + half) meet through shared memory
      float* b = buf[warp] + sub * p.lanes * 16;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (i0 + j * second < p.rot) {
          float4* d = reinterpret_cast<float4*>(b + i0 + j * second);
          d[0] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
          d[1] = make_float4(x[j][4], x[j][5], x[j][6], x[j][7]);
        }
      __syncwarp();
      if (isq || isk) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e0 = i0 + j * second;
          if (e0 >= p.rot) continue;
          if (half % 8 == 0) {  // a piece turns with a piece
            const bool first = e0 < half;
            const int j0 = first ? e0 : e0 - half;
            const float4* o = reinterpret_cast<const float4*>(b + (first ? e0 + half : e0 - half));
            const float4* c = reinterpret_cast<const float4*>(cs + j0);
            const float4* s = reinterpret_cast<const float4*>(sn + j0);
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 ov = o[i / 4], cv = c[i / 4], sv = s[i / 4];
              x[j][i] = fmaf(x[j][i], cv.x, first ? -ov.x * sv.x : ov.x * sv.x);
              x[j][i + 1] = fmaf(x[j][i + 1], cv.y, first ? -ov.y * sv.y : ov.y * sv.y);
              x[j][i + 2] = fmaf(x[j][i + 2], cv.z, first ? -ov.z * sv.z : ov.z * sv.z);
              x[j][i + 3] = fmaf(x[j][i + 3], cv.w, first ? -ov.w * sv.w : ov.w * sv.w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int e = e0 + i;
              if (e >= p.rot) break;
              const bool first = e < half;
              const int f = first ? e : e - half;
              const float o = b[first ? e + half : e - half];
              x[j][i] = fmaf(x[j][i], cs[f], first ? -o * sn[f] : o * sn[f]);
            }
          }
        }
      }
      if (isq) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (in[j])
            *reinterpret_cast<uint4*>(p.q + (r * p.Hq + hh) * p.D + i0 + j * second) =
                pack8(x[j], (const __nv_bfloat16*)nullptr);
      }
    }
    if (base + gpw > p.Hq) {  // some head of the warp is k or v
      const int h = isq ? 0 : isk ? hh - p.Hq : hh - p.Hq - p.Hk;
      const bool on[2] = {in[0] && !isq && keep, in[1] && !isq && keep};
      const float s = FMT == kFmtBf16 ? 0.f
                                      : scale_of<FMT == kFmtInt8 ? kFmtInt8 : kFmtFp8>(
                                            group_max(max(on[0] ? amax8(x[0]) : 0u, on[1] ? amax8(x[1]) : 0u), p.lanes));
      write_row<FMT>(x, i0, second, on, s, isk ? p.k : p.v, isk ? p.ks : p.vs, keep ? slot : 0, p.slots, h, p.Hk, p.D);
    }
  }
}

struct RowsArgs {
  const void *k, *v;  // rows given by the caller (write) / codes (read)
  void *ko, *vo;      // codes (write) / rows (read)
  const float *ksr, *vsr;
  float *ks, *vs;
  const int64_t* slot;
  int* err;
  int64_t T, slots, k_ld, k_lh, v_ld, v_lh;
  int Hk, D, lanes, vec;
};

// Quantises given K and V rows into their slots: a lane group per (token, kv head), K's and V's loads issued together.
// 65536 tokens x 8 x 128 bf16 -> int8: 79 us, 5.2 TB/s (0.79 of the copy rate); eight elements a lane and unpacked maxima
// took 140 us, bound by instructions.
template <int FMT, typename T>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const RowsArgs p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, gpw = 32 / p.lanes, i0 = (lane % p.lanes) * 8, second = p.lanes * 8;
  const uint32_t unit = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * gpw + lane / p.lanes;
  const int64_t t = unit / uint32_t(p.Hk);
  const int h = int(unit % uint32_t(p.Hk));
  const int64_t slot = t < p.T ? p.slot[t] : -1;
  if (slot >= p.slots && h == 0 && i0 == 0) record_error(p.err, kErrBadIndex);
  const bool keep = slot >= 0 && slot < p.slots;
  const bool on[2] = {keep && i0 < p.D, keep && i0 + second < p.D};
  Eight<T> e[2][2];  // [K, V][piece]
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    e[0][j].clear();
    e[1][j].clear();
    if (!on[j]) continue;
    e[0][j].load(reinterpret_cast<const T*>(p.k) + t * p.k_ld + h * p.k_lh + i0 + j * second, p.vec);
    e[1][j].load(reinterpret_cast<const T*>(p.v) + t * p.v_ld + h * p.v_lh + i0 + j * second, p.vec);
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const float s = scale_of<FMT>(group_max(max(e[kv][0].amax(), e[kv][1].amax()), p.lanes));
    float x[2][8];
    e[kv][0].get(x[0]);
    e[kv][1].get(x[1]);
    write_row<FMT>(x, i0, second, on, s, kv ? p.vo : p.ko, kv ? p.vs : p.ks, keep ? slot : 0, p.slots, h, p.Hk, p.D);
  }
}

// Reads cache rows back: a lane group per (token, kv head); a row without a slot (negative) is zeros. 65536 tokens x 8 x
// 128 int8 -> bf16: 65 us, 6.3 TB/s (0.96 of the copy rate).
template <int FMT, typename T>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const RowsArgs p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, gpw = 32 / p.lanes, i0 = (lane % p.lanes) * 8, second = p.lanes * 8;
  const uint32_t unit = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * gpw + lane / p.lanes;
  const int64_t t = unit / uint32_t(p.Hk);
  const int h = int(unit % uint32_t(p.Hk));
  if (t >= p.T) return;
  const int64_t slot = p.slot[t];
  if (slot >= p.slots && h == 0 && i0 == 0) record_error(p.err, kErrBadIndex);
  const bool keep = slot >= 0 && slot < p.slots;
  uint2 w[2][2] = {};  // [K, V][piece]
  float s[2] = {};
  if (keep) {
    const size_t at = (size_t(slot) * p.Hk + h) * p.D + i0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (i0 + j * second >= p.D) continue;
      w[0][j] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(p.k) + at + j * second);
      w[1][j] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(p.v) + at + j * second);
    }
    s[0] = p.ksr[size_t(h) * p.slots + slot];
    s[1] = p.vsr[size_t(h) * p.slots + slot];
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int kv = n / 2, j = n % 2;
    if (i0 + j * second >= p.D) continue;
    float x[8];
    decode4<FMT>(w[kv][j].x, x);
    decode4<FMT>(w[kv][j].y, x + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= s[kv];
    T* out = reinterpret_cast<T*>(kv ? p.vo : p.ko) + (t * p.Hk + h) * p.D + i0 + j * second;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(out) = pack8(x, out);
    }
  }
}

// Moves accepted rows (up to kMoveLayers attention layers at once). A block owns one column of ``pieces`` 16-byte pieces of
// one layer's K or V rows (or, in 8-bit caches, that layer's scales) for every move: it reads up to kThreads / pieces *
// kMovesPer moves' pieces, waits, and writes them, so a source is read before a later move overwrites it (an accepted
// path moves rows down onto positions that earlier moves have read), with no order between blocks needed. Bound by launch
// and two dependent loads at a round's few moves: columns are as wide as lets one pass hold all moves, 64 bytes at least.
// 16 layers of 4 x 256 bf16: 6 moves 2.0 us, 104 4.2 us, 832 24 us (4.5 TB/s through L2); with int8 rows 2.1, 3.2 and 15 us.
constexpr int kMovesPer = 4, kMoveLayers = 64, kMinPieces = 4, kMaxPieces = 32;
struct MoveTable {
  uint8_t* rows[kMoveLayers][2];
  float* scales[kMoveLayers][2];
};
__global__ void __launch_bounds__(kThreads)
kv_commit_kernel(const __grid_constant__ MoveTable tab, const int64_t* __restrict__ src, const int64_t* __restrict__ dst,
                 int n, int64_t slots, int row_bytes, int Hk, int pieces, int cols, int per_cache, int* err) {
  pdl_wait();
  pdl_trigger();
  const int l = blockIdx.x / (2 * per_cache), rest = blockIdx.x % (2 * per_cache);
  const int kv = rest / per_cache, col = rest % per_cache;
  const int step = kThreads / pieces, m0 = threadIdx.x / pieces, piece = threadIdx.x % pieces;
  int s[kMovesPer], d[kMovesPer];  // source and destination slot, negative: no move
  auto fetch = [&](int at) {
#pragma unroll
    for (int i = 0; i < kMovesPer; ++i) {
      const int m = at + i * step + m0;
      const int64_t from = m < n ? src[m] : -1, to = m < n ? dst[m] : -1;
      if (from >= slots || to >= slots) record_error(err, kErrBadIndex);
      const bool on = from >= 0 && to >= 0 && from < slots && to < slots && from != to;
      s[i] = on ? int(from) : -1;
      d[i] = int(to);
    }
  };
  fetch(0);
  for (int at = 0; at < n; at += step * kMovesPer) {
    int from[kMovesPer], to[kMovesPer];
#pragma unroll
    for (int i = 0; i < kMovesPer; ++i) from[i] = s[i], to[i] = d[i];
    fetch(at + step * kMovesPer);  // in flight with this pass
    if (col < cols) {
      uint8_t* base = tab.rows[l][kv];
      const int off = (col * pieces + piece) * 16;
      uint4 v[kMovesPer];
#pragma unroll
      for (int i = 0; i < kMovesPer; ++i)
        if (from[i] >= 0 && off < row_bytes) v[i] = *reinterpret_cast<const uint4*>(base + int64_t(from[i]) * row_bytes + off);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMovesPer; ++i)
        if (from[i] >= 0 && off < row_bytes) *reinterpret_cast<uint4*>(base + int64_t(to[i]) * row_bytes + off) = v[i];
    } else {
      float* base = tab.scales[l][kv];
      for (int h0 = 0; h0 < Hk; h0 += pieces) {
        const int h = h0 + piece;
        float v[kMovesPer];
#pragma unroll
        for (int i = 0; i < kMovesPer; ++i)
          if (from[i] >= 0 && h < Hk) v[i] = base[size_t(h) * slots + from[i]];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMovesPer; ++i)
          if (from[i] >= 0 && h < Hk) base[size_t(h) * slots + to[i]] = v[i];
      }
    }
    __syncthreads();
  }
}

int fmt_of(const torch::Tensor& t) {
  const auto ty = t.scalar_type();
  if (ty == at::kFloat8_e4m3fn) return kFmtFp8;
  if (ty == at::kChar) return kFmtInt8;
  TORCH_CHECK(ty == at::kBFloat16, "KV cache: the rows must be float8_e4m3fn, int8 or bfloat16");
  return kFmtBf16;
}

void check_cache(const char* who, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ks,
                 const torch::Tensor& vs, torch::Device dev) {
  TORCH_CHECK(k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.is_contiguous() &&
                  v.is_contiguous() && k.device() == dev && v.device() == dev,
              who, ": the K and V caches must be contiguous [slots, kv heads, head dim] of one type on the rows' device");
  const int fmt = fmt_of(k);
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0, who,
              ": the caches must start on a 16-byte boundary");
  TORCH_CHECK(k.size(2) >= 8 && k.size(2) <= 256 && k.size(2) % (fmt == kFmtBf16 ? 8 : 16) == 0, who,
              ": the head dim must be a multiple of 16 (8 in a bf16 cache) up to 256");
  if (fmt == kFmtBf16) return;
  for (const torch::Tensor* s : {&ks, &vs})
    TORCH_CHECK(s->defined() && s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == k.size(1) &&
                    s->size(1) == k.size(0) && s->is_contiguous() && s->device() == dev,
                who, ": the scales must be contiguous fp32 [kv heads, slots] on the rows' device");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

// Splits the projection's rows, normalises and rotates q and k by positions of several axes, writes K and V into 16-
// or 8-bit caches (a negative slot writes nothing) and returns q [T, Hq, D].
torch::Tensor prepare_axes(const torch::Tensor& qkv, const torch::Tensor& pos, const torch::Tensor& slot,
                           torch::Tensor kc, torch::Tensor vc, torch::Tensor ks, torch::Tensor vs,
                           const c10::optional<torch::Tensor>& qn, const c10::optional<torch::Tensor>& kn,
                           bool norm_offset, const torch::Tensor& inv, const std::vector<int64_t>& sections,
                           bool interleaved, int64_t Hq, int64_t rot, bool gated, double eps) {
  const at::cuda::CUDAGuard g(qkv.device());
  const char* who = "qkv_prepare";
  check_cache(who, kc, vc, ks, vs, qkv.device());
  const int64_t T = qkv.size(0), Hk = kc.size(1), D = kc.size(2);
  TORCH_CHECK(Hq > 0 && Hk > 0 && Hq * D < (int64_t(1) << 28), who, ": head counts must be positive");
  TORCH_CHECK(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 && qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 &&
                  aligned16(qkv.data_ptr()),
              who, ": the projection must be bf16 rows on 16-byte boundaries");
  TORCH_CHECK(qkv.size(1) == (Hq * (gated ? 2 : 1) + 2 * Hk) * D, who,
              ": the projection's columns do not match the heads");
  TORCH_CHECK(rot >= 0 && rot % 2 == 0 && rot <= D && inv.numel() >= rot / 2, who, ": rotary dims must be even, up to the head dim");
  TORCH_CHECK(pos.dim() == 2 && pos.size(1) == T && pos.scalar_type() == at::kLong && (pos.stride(1) == 1 || T == 1) &&
                  pos.size(0) >= 1 && pos.size(0) <= kMaxAxes && int64_t(sections.size()) == pos.size(0),
              who, ": positions must be int64 [axes, T], one section per axis, up to 4 axes");
  TORCH_CHECK(slot.dim() == 1 && slot.size(0) == T && slot.scalar_type() == at::kLong && slot.is_contiguous(), who,
              ": write slots must be contiguous int64 [T]");
  TORCH_CHECK(pos.device() == qkv.device() && slot.device() == qkv.device() && inv.device() == qkv.device() &&
                  inv.scalar_type() == at::kDouble && inv.is_contiguous(),
              who, ": positions and write slots must be on the projection's device");
  for (const auto* w : {&qn, &kn})
    TORCH_CHECK(!*w || ((*w)->device() == qkv.device() && (*w)->scalar_type() == at::kBFloat16 && (*w)->numel() == D && (*w)->is_contiguous() &&
                        aligned16((*w)->data_ptr())),
                who, ": q / k norm weights must be contiguous bf16 [head dim] on a 16-byte boundary");
  auto q = torch::empty({T, Hq, D}, qkv.options());
  if (T == 0) return q;
  PrepareArgs p = {};
  p.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.pos = pos.data_ptr<int64_t>();
  p.slot = slot.data_ptr<int64_t>();
  p.qn = qn ? reinterpret_cast<const __nv_bfloat16*>(qn->data_ptr()) : nullptr;
  p.kn = kn ? reinterpret_cast<const __nv_bfloat16*>(kn->data_ptr()) : nullptr;
  p.inv = inv.data_ptr<double>();
  p.k = kc.data_ptr();
  p.v = vc.data_ptr();
  const int fmt = fmt_of(kc);
  p.ks = fmt == kFmtBf16 ? nullptr : ks.data_ptr<float>();
  p.vs = fmt == kFmtBf16 ? nullptr : vs.data_ptr<float>();
  p.q = reinterpret_cast<__nv_bfloat16*>(q.data_ptr());
  p.err = gemm_error_word(qkv.device()).data_ptr<int>();
  p.slots = kc.size(0);
  p.ldq = qkv.stride(0);
  p.pos_ld = pos.stride(0);
  p.Hq = int(Hq);
  p.Hk = int(Hk);
  p.D = int(D);
  p.rot = int(rot);
  p.lanes = row_lanes(int(D));
  p.koff = int(Hq * D * (gated ? 2 : 1));
  p.axes = int(pos.size(0));
  for (int a = 0; a < p.axes; ++a) p.sec[a] = int(sections[a]);
  p.interleaved = interleaved;
  p.norm_offset = norm_offset;
  p.eps = float(eps);
  p.inv_d = 1.f / float(D);
  // A row's heads are spread over several blocks only while the rows alone leave SMs idle. One block a row / spread, us,
  // 24/4 x 256 into int8: 1 row 3.8 / 2.9, 128 rows 3.9 / 3.4, 512 6.3 / 6.3, 1024 9.8 / 11.1, 2048 17.6 / 20.5; 32/8 x 128
  // crosses at the same count.
  const int64_t passes = ceil_div(Hq + 2 * Hk, int64_t(kWarps) * (32 / p.lanes));
  const dim3 grid(T, T >= 512 ? 1 : passes);
  auto st = at::cuda::getCurrentCUDAStream().stream();
  if (fmt == kFmtFp8) C10_CUDA_CHECK(launch_pdl(prepare_axes_kernel<kFmtFp8>, grid, kThreads, 0, st, p));
  else if (fmt == kFmtInt8) C10_CUDA_CHECK(launch_pdl(prepare_axes_kernel<kFmtInt8>, grid, kThreads, 0, st, p));
  else C10_CUDA_CHECK(launch_pdl(prepare_axes_kernel<kFmtBf16>, grid, kThreads, 0, st, p));
  return q;
}

// Quantises rows k, v [T, Hk, D] (bf16, fp16 or fp32, any strides with contiguous elements) into their cache slots.
void kv_write(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& slot, torch::Tensor kc,
              torch::Tensor vc, torch::Tensor ks, torch::Tensor vs) {
  const at::cuda::CUDAGuard g(kc.device());
  const char* who = "kv_write";
  check_cache(who, kc, vc, ks, vs, k.device());
  const int fmt = fmt_of(kc);
  TORCH_CHECK(fmt != kFmtBf16, who, ": the cache must hold 8-bit rows");
  const int64_t T = k.size(0), Hk = kc.size(1), D = kc.size(2);
  const auto ty = k.scalar_type();
  TORCH_CHECK(k.dim() == 3 && k.sizes() == v.sizes() && v.scalar_type() == ty && v.device() == k.device() &&
                  k.size(1) == Hk && k.size(2) == D && k.stride(2) == 1 && v.stride(2) == 1,
              who, ": rows must be [T, kv heads, head dim] of one type, elements contiguous");
  TORCH_CHECK(ty == at::kBFloat16 || ty == at::kHalf || ty == at::kFloat, who, ": rows must be bf16, fp16 or fp32");
  TORCH_CHECK(slot.dim() == 1 && slot.size(0) == T && slot.scalar_type() == at::kLong && slot.is_contiguous() &&
                  slot.device() == k.device(),
              who, ": write slots must be contiguous int64 [T]");
  if (T == 0) return;
  RowsArgs p = {};
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.ko = kc.data_ptr();
  p.vo = vc.data_ptr();
  p.ks = ks.data_ptr<float>();
  p.vs = vs.data_ptr<float>();
  p.slot = slot.data_ptr<int64_t>();
  p.err = gemm_error_word(k.device()).data_ptr<int>();
  p.T = T;
  p.slots = kc.size(0);
  p.k_ld = k.stride(0);
  p.k_lh = k.stride(1);
  p.v_ld = v.stride(0);
  p.v_lh = v.stride(1);
  p.Hk = int(Hk);
  p.D = int(D);
  p.lanes = row_lanes(int(D));
  const int64_t item = k.element_size();
  p.vec = aligned16(p.k) && aligned16(p.v) && (p.k_ld * item) % 16 == 0 && (p.k_lh * item) % 16 == 0 &&
          (p.v_ld * item) % 16 == 0 && (p.v_lh * item) % 16 == 0;
  const int64_t blocks = ceil_div(T * Hk, int64_t(kWarps) * (32 / p.lanes));
  TORCH_CHECK(T * Hk < (int64_t(1) << 31), who, ": too many rows");
  auto st = at::cuda::getCurrentCUDAStream().stream();
#define E4_KV_WRITE(F, TY) C10_CUDA_CHECK(launch_pdl(kv_write_kernel<F, TY>, blocks, kThreads, 0, st, p))
#define E4_KV_TYPES(M, F)                          \
  if (ty == at::kBFloat16) M(F, __nv_bfloat16);    \
  else if (ty == at::kHalf) M(F, __half);          \
  else M(F, float)
  if (fmt == kFmtFp8) { E4_KV_TYPES(E4_KV_WRITE, kFmtFp8); } else { E4_KV_TYPES(E4_KV_WRITE, kFmtInt8); }
}

// The values of the cache rows at ``slot`` (negative: zeros) as [T, Hk, D] of ``dtype``.
std::vector<torch::Tensor> kv_read(const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& ks,
                                   const torch::Tensor& vs, const torch::Tensor& slot, at::ScalarType ty) {
  const at::cuda::CUDAGuard g(kc.device());
  const char* who = "kv_read";
  check_cache(who, kc, vc, ks, vs, slot.device());
  const int fmt = fmt_of(kc);
  TORCH_CHECK(fmt != kFmtBf16, who, ": the cache must hold 8-bit rows");
  TORCH_CHECK(ty == at::kBFloat16 || ty == at::kHalf || ty == at::kFloat, who, ": rows are read as bf16, fp16 or fp32");
  TORCH_CHECK(slot.dim() == 1 && slot.scalar_type() == at::kLong && slot.is_contiguous(), who,
              ": slots must be contiguous int64 [T]");
  const int64_t T = slot.size(0), Hk = kc.size(1), D = kc.size(2);
  auto o = kc.options().dtype(ty);
  auto k = torch::empty({T, Hk, D}, o), v = torch::empty({T, Hk, D}, o);
  if (T == 0) return {k, v};
  RowsArgs p = {};
  p.k = kc.data_ptr();
  p.v = vc.data_ptr();
  p.ko = k.data_ptr();
  p.vo = v.data_ptr();
  p.ksr = ks.data_ptr<float>();
  p.vsr = vs.data_ptr<float>();
  p.slot = slot.data_ptr<int64_t>();
  p.err = gemm_error_word(kc.device()).data_ptr<int>();
  p.T = T;
  p.slots = kc.size(0);
  p.Hk = int(Hk);
  p.D = int(D);
  p.lanes = row_lanes(int(D));
  const int64_t blocks = ceil_div(T * Hk, int64_t(kWarps) * (32 / p.lanes));
  TORCH_CHECK(T * Hk < (int64_t(1) << 31), who, ": too many rows");
  auto st = at::cuda::getCurrentCUDAStream().stream();
#define E4_KV_READ(F, TY) C10_CUDA_CHECK(launch_pdl(kv_read_kernel<F, TY>, blocks, kThreads, 0, st, p))
  if (fmt == kFmtFp8) { E4_KV_TYPES(E4_KV_READ, kFmtFp8); } else { E4_KV_TYPES(E4_KV_READ, kFmtInt8); }
  return {k, v};
}

// Moves rows src -> dst in every layer's caches, which have one type and shape: K and V rows [slots, ...] of any type,
// and in 8-bit caches the scales ``ks``, ``vs`` (else empty lists).
void kv_commit(const std::vector<torch::Tensor>& k, const std::vector<torch::Tensor>& v,
               const std::vector<torch::Tensor>& ks, const std::vector<torch::Tensor>& vs, const torch::Tensor& src,
               const torch::Tensor& dst) {
  const at::cuda::CUDAGuard g(src.device());
  const char* who = "kv_commit";
  const int64_t n = src.numel(), layers = int64_t(k.size());
  const bool quant = !ks.empty();
  TORCH_CHECK(src.scalar_type() == at::kLong && dst.scalar_type() == at::kLong && src.is_contiguous() &&
                  dst.is_contiguous() && dst.numel() == n && dst.device() == src.device() && n < (int64_t(1) << 31),
              who, ": moves must be contiguous int64 lists of one length on one device");
  TORCH_CHECK(v.size() == k.size() && ks.size() == (quant ? k.size() : 0) && vs.size() == ks.size(), who,
              ": one K and one V cache per layer");
  if (!n || !layers) return;
  int64_t slots = k[0].size(0);  // of the smallest cache: a move applies to every layer
  for (int64_t l = 0; l < layers; ++l) {
    if (quant) {
      check_cache(who, k[l], v[l], ks[l], vs[l], src.device());
      TORCH_CHECK(fmt_of(k[l]) != kFmtBf16, who, ": caches with scales must be 8-bit");
    }
    for (const torch::Tensor* t : {&k[l], &v[l]}) {
      TORCH_CHECK(t->dim() >= 2 && t->sizes().slice(1) == k[0].sizes().slice(1) && t->is_contiguous() &&
                      (!quant || t->size(0) == k[0].size(0)) && t->scalar_type() == k[0].scalar_type() &&
                      t->device() == src.device(),
                  who, ": the layers' caches must be contiguous, of one type and shape, on the moves' device");
      slots = std::min(slots, t->size(0));
      TORCH_CHECK(aligned16(t->data_ptr()), who, ": the caches must start on a 16-byte boundary");
    }
  }
  if (slots == 0) return;
  TORCH_CHECK(slots < (int64_t(1) << 31), who, ": too many slots");
  const int64_t row_bytes = k[0].numel() / k[0].size(0) * k[0].element_size(), Hk = quant ? k[0].size(1) : 0;
  TORCH_CHECK(row_bytes % 16 == 0 && row_bytes < (int64_t(1) << 30), who, ": a cache row must be a multiple of 16 bytes");
  int pieces = kMaxPieces;
  while (pieces > kMinPieces && kThreads / pieces * kMovesPer < n) pieces /= 2;
  const int cols = int(ceil_div(row_bytes, pieces * 16)), per_cache = cols + (quant ? 1 : 0);
  int* err = gemm_error_word(src.device()).data_ptr<int>();
  for (int64_t l0 = 0; l0 < layers; l0 += kMoveLayers) {
    const int64_t m = std::min<int64_t>(kMoveLayers, layers - l0);
    MoveTable tab = {};
    for (int64_t l = 0; l < m; ++l) {
      tab.rows[l][0] = reinterpret_cast<uint8_t*>(k[l0 + l].data_ptr());
      tab.rows[l][1] = reinterpret_cast<uint8_t*>(v[l0 + l].data_ptr());
      if (!quant) continue;
      tab.scales[l][0] = ks[l0 + l].data_ptr<float>();
      tab.scales[l][1] = vs[l0 + l].data_ptr<float>();
    }
    C10_CUDA_CHECK(launch_pdl(kv_commit_kernel, m * 2 * per_cache, kThreads, 0,
                              at::cuda::getCurrentCUDAStream().stream(), tab, src.data_ptr<int64_t>(),
                              dst.data_ptr<int64_t>(), int(n), slots, int(row_bytes), int(Hk), pieces, cols, per_cache,
                              err));
  }
}

}  // namespace e4
