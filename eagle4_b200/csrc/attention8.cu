// Tree attention over a paged 8-bit KV cache (e4m3 or int8 codes, one fp32 scale per token and kv head).
//
// Every query row attends to a *logical key sequence*: the committed context positions [ctx_start, ctx_len) of its
// request (through the block table), then up to 128 extra physical slots (its tree ancestors and itself). With key
// codes k, value codes v and their scales a, b the row's output is
//     o = sum_j p_j b_j v_j / sum_j p_j,   p_j = exp(scale a_j (q . k_j) - max).
//
// The codes go to the tensor cores as they lie in the cache; no 8-bit value is ever widened. What is not 8-bit is
// cut into 8-bit digits instead: q and the weights p_j b_j become three digits each (e4m3: the rounded value, then
// the remainder times 16, twice: within 2^-12 of the value down to 2^-14 of full scale, within 2^-26 of full scale below;
// int8: signed base-256 digits of a fixed-point number, within 2^-23 of full scale), one MMA column per digit, and the three products are added in fp32 afterwards. The tensor cores are idle most of the
// time at these sizes, so three columns cost nothing, and the operands need half the shared memory and no conversion
// work per key. The value scale goes into the softmax: u_j = score_j log2(e) + log2(b_j) is what the running maximum
// is taken over, so the weights w_j = 2^(u_j - max u) = p_j b_j lie in (0, 1] whatever the scales are, which is what
// their digits need; the softmax's sum takes w_j / b_j.
//
// Work: the keys of every (row, kv head) are cut into 128-key chunks counted from ctx_start; all chunks of all rows
// form one list that a persistent grid divides evenly, so ragged batches and single long rows both fill the GPU. Four
// warps stream K and V rows (and scales) of the CTA's chunks through a ring of shared-memory stages with 16-byte
// asynchronous copies straight into the 128-byte-swizzled UMMA layouts; four more (head dims over 128: eight, half of the
// heads each) and one that issues the MMAs run
//   S^T[key, column] = K . Q^T      (M = 128 keys, N = 3 digits x heads, K = D)
//   weights, digits -> shared memory
//   O^T[d, column] = V^T . W^T      (M = 128 head dims, V as an MN-major operand, K = 128 keys)
// and fold each chunk's (maximum, sum, output) into fp32 registers. A (row, kv head) inside one CTA is finished there;
// one cut by a CTA boundary leaves partials that a small second kernel folds.
//
// Bound: HBM for long caches (32 rows of 32768 keys, 8 x 128: 420 us, 5.3 TB/s, 0.81 of the copy rate; one row of 131071
// keys, 4 x 256 int8: 58 us, 0.72); the softmax warps' instructions, some 2000 cycles a chunk, where rows are short or
// share their keys through L2 (8 x 16 tree rows over 1900 keys: 118 us; a prompt of 8192 rows, 4 x 256: 16.8 ms); launch
// and the dependent loads of two kernels for one short row (4096 keys: 14 us). Three digits instead of two cost nothing measurable and keep the
// digits' error at or below the rounding of fp16 outputs.
//
// A row's result must not depend on its batch: a token decoded alone and the same token verified inside a tree have to
// agree bit for bit. So the order of folding is fixed by the row's key count alone: a row's chunks are folded in order
// within pieces of ``piece_chunks`` chunks (so sized that one row alone spreads over the whole GPU), and the pieces in
// order. CTA boundaries fall between pieces. A CTA that holds all pieces of a row folds them in registers, with the
// same operations the second kernel uses otherwise.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "quant.cuh"

namespace e4 {

torch::Tensor gemm_error_word(torch::Device dev);

namespace {

constexpr int kChunk = 128;    // logical keys per chunk: the MMA's M
constexpr int kLoad = 128;     // threads that load
// Threads for softmax and output, before the loading ones and the warp that issues the MMAs (an issue takes some 90
// cycles, too much for a warp the others wait for): one group of 128 up to head dim 128, where two CTAs share an SM (up
// to 8 heads); two with half of the heads each above, where one CTA has the SM and a chunk's output is twice as long.
// Measured when it was tried: two groups at head dim 128 need 500 us for 32 x 32768 keys where one needed 400 (twice the
// waiting threads, the same work).
__host__ __device__ constexpr int math_threads(int KB) { return KB * 128; }
__host__ __device__ constexpr int num_threads(int KB) { return math_threads(KB) + kLoad + 32; }
constexpr int kTerms = 3;      // 8-bit digits per 16-bit query or weight
constexpr int kMaxExtra = 128;

struct Args {
  const void* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *bt, *req, *start, *end, *extra, *n_extra;
  const void* gate;
  void* out;
  float* ws;    // partials: [CTA boundary][piece][G][D + 4]; a (row, kv head) lies with the first boundary that cuts it
  int4* info;   // per CTA: (row, head, piece, the row's chunks) where its work begins (an empty one: the next one's)
  int* err;
  int64_t slots, ldg;
  int T, Hq, Hk, G, D, page, bt_ld, bt_rows, extra_ld, max_chunks, area, spread, fp16;
  float scale;  // times log2(e)
};

E4_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
E4_DEV float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
E4_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
E4_DEV float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

E4_DEV void cp16(uint32_t dst, const void* src, bool on) {  // zero-fills when off
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
E4_DEV void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
E4_DEV void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
// This thread's earlier cp.async copies arrive on ``bar`` (counted in its initial count) when they have landed.
E4_DEV void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
E4_DEV void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Waits for the phase with ``parity``; false after about two seconds. The SM's own clock bounds it: reading the global
// timer in the loop costs more than most of these waits last.
E4_DEV bool spin_wait(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > (1ll << 32)) return false;
  return true;
}

// Shared-memory descriptor of an MN-major 8-bit tile with the 128-byte swizzle: 128 M elements per row, 8-row (K)
// groups 1024 bytes apart; one atom covers M = 128, so the leading offset is not used.
E4_DEV uint64_t sdesc_mn8(uint32_t saddr) {
  uint64_t d = 0;
  d |= uint64_t((saddr & 0x3FFFFu) >> 4);
  d |= uint64_t(1) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}

// True in one lane of a converged warp. The issue loop's thread is chosen by this, not by its lane number: the compiler
// then knows that one lane runs, and products inside data-dependent branches stay right (chosen by ``lane == 0``, a
// condition around each product gave wrong sums).
E4_DEV bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(on));
  return on != 0;
}

// D[tmem] (+)= A[smem] . B[smem]^T on 8-bit operands: e4m3 with fp32 sums, or int8 with int32 sums.
template <int FMT>
E4_DEV void umma8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (FMT == kFmtFp8)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Instruction descriptor: e4m3 x e4m3 -> fp32, or s8 x s8 -> s32; ``a_mn``: A is MN-major.
template <int FMT>
E4_DEV uint32_t idesc8(int N, bool a_mn) {
  const uint32_t types = FMT == kFmtFp8 ? (1u << 4) : ((2u << 4) | (1u << 7) | (1u << 10));
  return types | (a_mn ? 1u << 15 : 0u) | (uint32_t(N >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

// N consecutive 32-bit columns of this thread's TMEM lane, without the wait.
template <int N>
E4_DEV void tmem_ld(uint32_t t, uint32_t* r) {
  if constexpr (N == 2)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(t));
  else if constexpr (N == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(t));
  else if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(t));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(t));
}
E4_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------------- digits
// Three digits of x (|x| <= 1 times the format's full scale) for a pair of numbers, in the low two bytes of d (the
// first number's lowest; the upper bytes are not defined), and the sum of three products.
template <int FMT>
struct Digits;

template <>
struct Digits<kFmtFp8> {
  static constexpr int kExp = 8;  // full scale 2^8 (e4m3 reaches 448)
  E4_DEV static void cut2(float x, float y, uint32_t* d) {
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
      const __nv_fp8x2_storage_t c = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
      d[t] = c;
      if (t + 1 < kTerms) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3)));
        x = (x - f.x) * 16.f;
        y = (y - f.y) * 16.f;
      }
    }
  }
  E4_DEV static float join(uint32_t a, uint32_t b, uint32_t c) {
    return fmaf(fmaf(__uint_as_float(c), 0.0625f, __uint_as_float(b)), 0.0625f, __uint_as_float(a));
  }
};

template <>
struct Digits<kFmtInt8> {
  static constexpr int kExp = 22;  // full scale 2^22: the top digit stays within +-64
  // signed base-256 digits: adding 0x8080 makes every carry, flipping the low digits' top bits takes it back
  E4_DEV static uint32_t cut(float x) { return uint32_t(__float2int_rn(x) + 0x8080) ^ 0x8080u; }
  E4_DEV static void cut2(float x, float y, uint32_t* d) {
    const uint32_t a = cut(x), b = cut(y);
    d[0] = __byte_perm(a, b, 0x0062);
    d[1] = __byte_perm(a, b, 0x0051);
    d[2] = __byte_perm(a, b, 0x0040);
  }
  // |b|, |c| <= 128 * 128 * 256 = 2^22: b * 256 + c fits in 32 bits
  E4_DEV static float join(uint32_t a, uint32_t b, uint32_t c) {
    return fmaf(float(int(a)), 65536.f, float(int(b) * 256 + int(c)));
  }
};

E4_DEV float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// ------------------------------------------------------------------------------------------------------- layout
// The rings of K tiles (with the stage's 128 + 128 scales) and V tiles, and the CTA's dynamic shared memory.
constexpr int kStages = 3;
__host__ __device__ constexpr int columns(int NH) { return (kTerms * NH + 15) / 16 * 16; }
__host__ __device__ constexpr int smem_bytes(int KB, int NH) {
  // from a 1024-byte boundary on: K and V tiles, then Q [KB][columns][128], two W [columns][128], then the scales
  return kStages * (2 * KB * kChunk * 128 + 2 * kChunk * 4) + (KB + 2) * columns(NH) * 128;
}
// CTAs that share an SM: two need 2 x (dynamic + 2048 static + 1024 reserved) bytes within its 228 KB and 96 registers a
// thread. With 5 to 8 heads the two fit to the byte and spill some 200 bytes a thread: 32 rows of 32768 keys, 64/8 heads x
// 128, take 640 us (fp8) and 646 us (int8), one CTA without spills 642 and 768.
__host__ __device__ constexpr int ctas_per_sm(int KB, int NH) { return KB == 1 && NH <= 8 ? 2 : 1; }
static_assert(ctas_per_sm(1, 8) * (smem_bytes(1, 8) + 2048 + 1024) <= 228 * 1024, "two CTAs an SM up to 8 heads");
// S and O accumulators, two of each
__host__ __device__ constexpr int tmem_columns(int KB, int NH) {
  int n = 32;
  while (n < 2 * (KB + 1) * columns(NH)) n *= 2;
  return n;
}

// A row's context positions, for any two int32 bounds.
E4_DEV int context_keys(const Args& p, int r) {
  const int a = p.start[r], b = p.end[r];
  return b > a ? int(min(uint32_t(b) - uint32_t(a), 0x7fffffffu)) : 0;
}
E4_DEV int total_keys(const Args& p, int r) {
  const uint32_t n = uint32_t(context_keys(p, r)) + uint32_t(min(max(p.n_extra[r], 0), p.extra_ld));
  if (n > uint32_t(p.max_chunks * kChunk)) {  // (at most 2^31 - 256: checked on the host)
    record_error(p.err, kErrBadShape);
    return p.max_chunks * kChunk;
  }
  return int(n);
}
// Chunks of a piece of a row with ``n`` chunks: its pieces over all kv heads come to about ``spread``.
E4_DEV int piece_chunks(const Args& p, int n) { return max((n * p.Hk + p.spread - 1) / p.spread, 1); }

// (M, L) and one output element folded: maxima in log2 units.
struct Fold {
  float a, b;
};
E4_DEV Fold fold_stats(float& M, float& L, float m, float l) {
  const float n = fmaxf(M, m);
  Fold f = {ex2(M - n), ex2(m - n)};
  L = fmaf(l, f.b, __fmul_rn(L, f.a));
  M = n;
  return f;
}
E4_DEV float fold(float A, float o, Fold f) { return fmaf(o, f.b, __fmul_rn(A, f.a)); }

E4_DEV void store_out(const Args& p, int r, int qh, int d, float A, float L) {
  float x = L == 0.f ? 0.f : A / L;
  const size_t at = (size_t(r) * p.Hq + qh) * p.D + d;
  if (p.fp16) {
    if (p.gate) x *= sigmoidf_(__half2float(reinterpret_cast<const __half*>(p.gate)[r * p.ldg + qh * p.D + d]));
    reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(x);
  } else {
    if (p.gate) x *= sigmoidf_(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.gate)[r * p.ldg + qh * p.D + d]));
    reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(x);
  }
}
E4_DEV void store_zero(const Args& p, int r, int i) {
  const size_t at = size_t(r) * p.Hq * p.D + i;
  reinterpret_cast<uint16_t*>(p.out)[at] = 0;
}
E4_DEV float load_q(const Args& p, size_t at) {
  return p.fp16 ? __half2float(reinterpret_cast<const __half*>(p.q)[at])
                : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[at]);
}

// A walk over chunks in order: rows, kv heads, chunks.
struct Walk {
  int r, h, c, n, total, piece;
  E4_DEV void next(const Args& p) {
    if (++c < n) return;
    next_head(p);
  }
  E4_DEV void next_head(const Args& p) {
    c = 0;
    if (++h < p.Hk) return;
    h = 0;
    seek(p, r + 1);
  }
  E4_DEV void seek(const Args& p, int row) {  // the first row from ``row`` on that has keys
    for (r = row; r < p.T; ++r) {
      total = total_keys(p, r);
      n = (total + kChunk - 1) / kChunk;
      if (n) break;
    }
    piece = piece_chunks(p, n);
  }
};

// Sums of NH values over the warp: the lanes halve the values among them while they halve the lanes they still have to
// add (NH / 2 + NH / 4 + ... + 1 + log2(32 / NH) shuffles). Lane l ends with value l / (32 / NH).
template <int NH>
E4_DEV float warp_sums(float* v, int lane) {
  int n = NH;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool up = lane & o;
#pragma unroll
      for (int j = 0; j < NH / 2; ++j) {
        if (j < n) {
          const float give = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
          v[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

// What a thread keeps of a row's fold for its H heads, at KB head dims: the running piece and the row so far.
template <int H, int KB>
struct State {
  float gM[H], gL[H], gA[KB][H], rM[H], rL[H], rA[KB][H];
  int region, part, in_piece;  // where its partials go: the first boundary that cuts it (less one), the piece
  bool whole;  // this CTA holds all of the row's chunks
  E4_DEV void clear_piece() {
    in_piece = 0;
#pragma unroll
    for (int g = 0; g < H; ++g) {
      gM[g] = -INFINITY;
      gL[g] = 0.f;
#pragma unroll
      for (int b = 0; b < KB; ++b) gA[b][g] = 0.f;
    }
  }
  E4_DEV void clear_row() {
#pragma unroll
    for (int g = 0; g < H; ++g) {
      rM[g] = -INFINITY;
      rL[g] = 0.f;
#pragma unroll
      for (int b = 0; b < KB; ++b) rA[b][g] = 0.f;
    }
  }
};

// Takes a finished piece into the row, or out as a partial; writes the row when it is finished. Heads [g0, g0 + H).
template <int H, int KB>
E4_DEV void end_piece(const Args& p, const Walk& f, State<H, KB>& s, int g0, int t, bool last) {
  if (!s.whole) {
    if (s.part >= p.area || s.region + 1 >= gridDim.x) {
      record_error(p.err, kErrBadShape);
    } else {
      float* ws = p.ws + ((size_t(s.region) * p.area + s.part) * p.G + g0) * (p.D + 4);
#pragma unroll
      for (int g = 0; g < H; ++g) {
        if (g0 + g >= p.G) break;
#pragma unroll
        for (int b = 0; b < KB; ++b)
          if (b * 128 + t < p.D) ws[g * (p.D + 4) + b * 128 + t] = s.gA[b][g];
        if (t == 0) {
          ws[g * (p.D + 4) + p.D] = s.gM[g];
          ws[g * (p.D + 4) + p.D + 1] = s.gL[g];
        }
      }
    }
    ++s.part;
  } else {
#pragma unroll
    for (int g = 0; g < H; ++g) {
      const Fold r = fold_stats(s.rM[g], s.rL[g], s.gM[g], s.gL[g]);
#pragma unroll
      for (int b = 0; b < KB; ++b) s.rA[b][g] = fold(s.rA[b][g], s.gA[b][g], r);
    }
    if (last) {
#pragma unroll
      for (int g = 0; g < H; ++g) {
        if (g0 + g >= p.G) break;
#pragma unroll
        for (int b = 0; b < KB; ++b)
          if (b * 128 + t < p.D) store_out(p, f.r, f.h * p.G + g0 + g, b * 128 + t, s.rA[b][g], s.rL[g]);
      }
    }
  }
  s.clear_piece();
}

// ------------------------------------------------------------------------------------------------------- kernel
template <int FMT, int NH, int KB>
__global__ void __launch_bounds__(num_threads(KB), ctas_per_sm(KB, NH)) attn8_kernel(const Args p) {
  constexpr int NC = columns(NH), NS = kStages, kTile = kChunk * 128, kTmem = tmem_columns(KB, NH);
  constexpr int kMath = math_threads(KB), kThreads = num_threads(KB), H = NH / KB;  // H: heads per thread
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS], q_full, w_full[2], s_done[2], o_done[2];
  __shared__ uint32_t tmem_holder;
  __shared__ int s_warp[kThreads / 32], s_at[2][4];  // begin and end: row, head, chunk, position
  __shared__ __align__(16) float red_m[2][4][NH], red_l[2][4][NH], s_qf[NH];
  __shared__ __align__(16) int s_cell[kLoad / 32][32];
  __shared__ int s_bad, s_first;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* Vs = smem + NS * KB * kTile;
  unsigned char* Qt = smem + NS * 2 * KB * kTile;
  unsigned char* Ws = Qt + KB * NC * 128;
  float* scales = reinterpret_cast<float*>(Ws + 2 * NC * 128);  // [stage][K 128 | V 128]

  if (tid == 32) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], kLoad);
      mbar_init(&v_full[i], kLoad);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&q_full, 1);
    for (int i = 0; i < 2; ++i) {  // two of each: a thread may wait for one product while the next completes
      mbar_init(&w_full[i], kMath);
      mbar_init(&s_done[i], 1);
      mbar_init(&o_done[i], 1);
    }
    mbar_fence_init();
    s_bad = 0;
  }
  // columns without a head and head dims past D stay zero
  for (int i = tid; i < (KB + 2) * NC * 8; i += kThreads) reinterpret_cast<uint4*>(Qt)[i] = make_uint4(0, 0, 0, 0);
  if (p.D < KB * 128)
    for (int i = tid; i < NS * 2 * KB * kTile / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  // TMEM is taken after the kernel before has ended and before the next one may start: two kernels on one SM that each
  // hold some of it, one waiting for the other, would wait for good.
  pdl_wait();
  if (warp == 0) tmem_alloc(&tmem_holder, kTmem);

  // chunks of all rows and heads: a block-wide prefix sum, a run of rows per thread
  const int per = (p.T + kThreads - 1) / kThreads;
  int mine = 0;
  for (int r = tid * per; r < min(p.T, (tid + 1) * per); ++r) mine += (total_keys(p, r) + kChunk - 1) / kChunk * p.Hk;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (tid < 2) {
    s_at[tid][0] = p.T;
    s_at[tid][1] = s_at[tid][2] = 0;
    s_at[tid][3] = -1;
  }
  __syncthreads();
  pdl_trigger();
  int chunks = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = chunks;
    chunks += s_warp[w];
  }
  // this CTA begins and ends at the first piece from its even share's bounds on
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = int(int64_t(chunks) * (blockIdx.x + e) / gridDim.x);
    int base = before + incl - mine;
    if (x < base || x >= base + mine) continue;
    for (int r = tid * per;; ++r) {
      const int n = (total_keys(p, r) + kChunk - 1) / kChunk;
      if (x < base + n * p.Hk) {
        const int h = (x - base) / n, ps = piece_chunks(p, n);
        const int c = min(((x - base) % n + ps - 1) / ps * ps, n);
        s_at[e][0] = r;
        s_at[e][1] = h;
        s_at[e][2] = c;
        s_at[e][3] = base + h * n + c;
        break;
      }
      base += n * p.Hk;
    }
  }
  __syncthreads();
  Walk w = {};
  w.seek(p, s_at[0][0]);
  w.h = s_at[0][1];
  w.c = s_at[0][2];
  if (w.r < p.T && w.c == w.n) w.next_head(p);
  if (tid == 0) {
    p.info[blockIdx.x] = make_int4(w.r, w.h, w.c / w.piece, w.n);
    // The boundary before CTA b lies at chunk floor(chunks b / grid): the first one past the start of the (row, kv head)
    // that this CTA begins inside of (read after the softmax warps' first barrier).
    s_first = w.c ? int((int64_t(s_at[0][3] - w.c + 1) * gridDim.x + chunks - 1) / chunks) - 1 : 0;
  }
  const int end = s_at[1][3] < 0 ? chunks : s_at[1][3];
  const int count = s_at[0][3] < 0 ? 0 : end - s_at[0][3];  // chunks of this CTA
  for (int r = blockIdx.x; r < p.T; r += gridDim.x)  // rows that see nothing
    if (total_keys(p, r) == 0)
      for (int i = tid; i < p.Hq * p.D; i += kThreads) store_zero(p, r, i);

  // A wait that runs out records its error; every later wait of the CTA is then skipped, so the CTA ends (with a wrong
  // result and the error word set) instead of spinning.
  auto wait1 = [&](uint64_t* bar, uint32_t parity, int code) {  // one thread
    if (!*reinterpret_cast<volatile int*>(&s_bad) && !spin_wait(bar, parity)) {
      record_error(p.err, code);
      s_bad = 1;
    }
  };
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {  // a warp
    wait1(bar, parity, code);
    __syncwarp();
  };

  if (warp == kMath / 32 + kLoad / 32) {
    // ---- MMAs, by one thread: S(i + 1) before O(i) where both have the same query. Waiting for w_full(i) also says that
    // S(i) and its scales have been read and O(i - 2) folded, so the buffers of S(i + 2) and O(i) are free. Head dims
    // past D are zeros in both operands: all products are issued, whatever D is.
    if (elect_one()) {
      tc_fence_after();
      const uint32_t tmem = tmem_holder, id_s = idesc8<FMT>(NC, false), id_o = idesc8<FMT>(NC, true);
      const uint32_t kt = smem_u32(smem), vt = smem_u32(Vs), qt = smem_u32(Qt), wt = smem_u32(Ws);
      int heads = 0;  // (row, kv head)s begun
      auto issue_s = [&](int i, bool begins) {
        if (begins) wait1(&q_full, heads++ & 1, kErrTimeoutMma);
        wait1(&k_full[i % NS], (i / NS) & 1, kErrTimeoutProducer);
        fence_async_smem();  // the copies landed through the generic proxy
        tc_fence_after();
        const uint64_t a = sdesc_sw128(kt + (i % NS) * KB * kTile), b = sdesc_sw128(qt);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma8<FMT>(tmem + (i & 1) * NC, a + (kb * kTile + ks * 32) / 16, b + (kb * NC * 128 + ks * 32) / 16, id_s,
                       (kb | ks) != 0);
        umma_commit(&s_done[i & 1]);
      };
      if (count) issue_s(0, true);
      for (int i = 0; i < count; ++i) {
        const int st = i % NS;
        w.next(p);
        const bool more = i + 1 < count, begins = w.c == 0;
        if (more && !begins) issue_s(i + 1, false);
        wait1(&w_full[i & 1], (i >> 1) & 1, kErrTimeoutMma);
        wait1(&v_full[st], (i / NS) & 1, kErrTimeoutProducer);
        mbar_arrive(&k_empty[st]);
        fence_async_smem();
        tc_fence_after();
        const uint64_t a = sdesc_mn8(vt + st * KB * kTile), b = sdesc_sw128(wt + (i & 1) * NC * 128);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma8<FMT>(tmem + 2 * NC + ((i & 1) * KB + kb) * NC, a + (kb * kTile + ks * 4096) / 16, b + ks * 32 / 16, id_o,
                       ks != 0);
        umma_commit(&o_done[i & 1]);
        if (i + NS < count) umma_commit(&v_empty[st]);  // (a load waits for it)
        if (more && begins) issue_s(i + 1, true);
      }
    }
    __syncwarp();
  } else if (warp >= kMath / 32) {
    // ---- loads: a warp copies 32 keys of every chunk; a row is LPR lanes of 16 bytes, and each of the 32 / LPR groups
    // of lanes takes kPass rows in order. The keys' rows meet their lanes through shared memory, four a load: issue
    // slots of the load unit are what this warp spends most.
    constexpr int LPR = KB * 8, kPass = LPR;
    const int lw = warp - kMath / 32, piece = lane % LPR, key = lw * 32 + lane, r0 = lane / LPR * kPass;
    const bool in = piece * 16 < p.D;
    const uint32_t smem0 = smem_u32(smem), scale0 = smem_u32(scales);
    const uint32_t dst0 = uint32_t(piece / 8) * kTile + uint32_t(lw * 32 + r0) * 128;
    // this lane's key of a chunk: its page-table entry and place in the page, or its extra slot
    int entry = -1, rest = 0, row = -1, c0 = 0, nctx = 0;
    const int* table = nullptr;  // the row's block-table row (null: no such request)
    enum { kNone, kPage, kExtra, kBad } kind = kNone;
    const int shift = (p.page & (p.page - 1)) == 0 ? __ffs(p.page) - 1 : -1;
    auto look = [&]() {
      if (w.r != row) {
        row = w.r;
        c0 = p.start[row];
        nctx = context_keys(p, row);
        const int b = p.req[row];
        table = b >= 0 && b < p.bt_rows ? p.bt + int64_t(b) * p.bt_ld : nullptr;
      }
      const int kk = w.c * kChunk + key;
      kind = kNone;
      if (kk >= w.total) return;
      // the entry is not looked at before the next chunk's turn: nothing here waits for it
      const int pos = c0 + kk, blk = shift >= 0 ? pos >> shift : pos / p.page;
      const int* from = p.extra + int64_t(w.r) * p.extra_ld + (kk - nctx);
      kind = kExtra;
      if (kk < nctx) {
        rest = pos - blk * p.page;
        kind = table && pos >= 0 && blk < p.bt_ld ? kPage : kBad;
        from = kind == kPage ? table + blk : nullptr;
      }
      if (from) entry = __ldg(from);
    };
    if (count) look();
    for (int i = 0; i < count; ++i) {
      const int st = i % NS;
      int64_t slot = -1;
      if (kind == kExtra) slot = entry;
      if (kind == kPage) slot = entry < 0 ? -1 : int64_t(entry) * p.page + rest;
      if (kind != kNone && (slot < 0 || slot >= p.slots)) {
        record_error(p.err, kErrBadIndex);
        slot = -1;
      }
      const int64_t so = slot < 0 ? 0 : w.h * p.slots + slot;
      __syncwarp();
      s_cell[lw][lane] = slot < 0 ? -1 : int(slot) * p.Hk + w.h;  // (slots * Hk < 2^31)
      const bool all = __all_sync(0xffffffffu, slot >= 0);
      w.next(p);
      if (i + 1 < count) look();  // the next chunk's entries arrive while this one's copies are issued
      __syncwarp();  // the lanes' cells are written before others read them
      int64_t src[kPass];
#pragma unroll
      for (int n = 0; n < kPass; n += 4) {
        const int4 c = *reinterpret_cast<const int4*>(&s_cell[lw][r0 + n]);
        src[n] = int64_t(c.x) * p.D;
        src[n + 1] = int64_t(c.y) * p.D;
        src[n + 2] = int64_t(c.z) * p.D;
        src[n + 3] = int64_t(c.w) * p.D;
      }
      auto copy = [&](uint32_t tile, const uint8_t* from) {
        if (!in) return;
        if (all) {
#pragma unroll
          for (int n = 0; n < kPass; ++n)
            cp16(tile + dst0 + n * 128 + ((uint32_t(piece & 7) ^ (n & 7)) << 4), from + src[n]);
        } else {
#pragma unroll
          for (int n = 0; n < kPass; ++n)
            cp16(tile + dst0 + n * 128 + ((uint32_t(piece & 7) ^ (n & 7)) << 4), src[n] < 0 ? from : from + src[n],
                 src[n] >= 0);
        }
      };
      if (i >= NS) wait(&k_empty[st], (i / NS - 1) & 1, kErrTimeoutProducer);
      copy(smem0 + st * KB * kTile, p.k + piece * 16);
      cp4(scale0 + (st * 2 * kChunk + key) * 4, p.ks + so, slot >= 0);
      cp4(scale0 + (st * 2 * kChunk + kChunk + key) * 4, p.vs + so, slot >= 0);
      cp_arrive(&k_full[st]);
      if (i >= NS) wait(&v_empty[st], (i / NS - 1) & 1, kErrTimeoutProducer);
      copy(smem0 + (NS + st) * KB * kTile, p.v + piece * 16);
      cp_arrive(&v_full[st]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- softmax, output: thread t of a group is key t of the chunk, then head dim t (and t + 128) of the output; a
    // second group has heads [H, 2 H). Heads past G compute on zero columns and are never stored.
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    const int G = p.G, t = tid & 127, quad = warp & 3, wg = warp >> 2, g0 = KB == 1 ? 0 : wg * H;
    const uint32_t lanes = tmem + (uint32_t(quad * 32) << 16) + g0;
    State<H, KB> s;
    float m[H], pm[H];  // maxima of this chunk and the one before
    // One step takes chunk i to its weights, then folds the output of chunk i - 1, whose product ran meanwhile.
    Walk f = w;  // the chunk being folded
    for (int i = 0; i <= count; ++i) {
      const int st = i % NS;
      if (i < count) {
        if (i == 0 || w.c == 0) {  // a (row, kv head) begins
          // the kv head's query heads: a full-scale power of two per head, digits into Q's columns (digit-major)
          named_bar(3, kMath);  // the last head's factors have been read
          for (int g = warp; g < NH; g += kMath / 32) {
            const size_t at = (size_t(w.r) * p.Hq + w.h * G + g) * p.D;
            float x[KB * 4];
            float am = 0.f;
#pragma unroll
            for (int j = 0; j < KB * 4; ++j) {
              const int d = lane * 4 + (j & 3) + (j >> 2) * 128;
              x[j] = g < G && d < p.D ? load_q(p, at + d) : 0.f;
              am = max_nan(am, fabsf(x[j]));
            }
            am = warp_max_nan(am);
            const int e = max(int(__float_as_uint(am) >> 23) - 127, -100);
            const float up = pow2f(Digits<FMT>::kExp - 1 - e), down = pow2f(e - Digits<FMT>::kExp + 1);
#pragma unroll
            for (int jj = 0; jj < KB; ++jj) {
              uint32_t a[kTerms], b[kTerms];
              Digits<FMT>::cut2(x[jj * 4] * up, x[jj * 4 + 1] * up, a);
              Digits<FMT>::cut2(x[jj * 4 + 2] * up, x[jj * 4 + 3] * up, b);
#pragma unroll
              for (int n = 0; n < kTerms; ++n) {
                const int col = n * NH + g, b16 = lane >> 2;
                *reinterpret_cast<uint32_t*>(Qt + jj * NC * 128 + col * 128 + ((b16 ^ (col & 7)) * 16) + (lane & 3) * 4) =
                    __byte_perm(a[n], b[n], 0x5410);
              }
            }
            // a query with a NaN or an infinity makes every score NaN
            if (lane == 0) s_qf[g] = am < INFINITY ? down * p.scale : __int_as_float(0x7fffffff);
          }
          fence_async_smem();
          named_bar(3, kMath);
          if (tid == 0) mbar_arrive(&q_full);
        }
        wait(&k_full[st], (i / NS) & 1, kErrTimeoutProducer);
        const float ksc = scales[st * 2 * kChunk + t], vsc = scales[st * 2 * kChunk + kChunk + t];
        const bool live = w.c * kChunk + t < w.total;
        const float vse = vsc < kScaleFloor ? kScaleFloor : vsc;  // keeps NaN
        const float lv = lg2(vse), iv = live ? __fdividef(1.f, vse) : 0.f;
        wait(&s_done[i & 1], (i >> 1) & 1, kErrTimeoutMma);
        tc_fence_after();
        float u[H];
        {
          uint32_t d[kTerms][H];
#pragma unroll
          for (int n = 0; n < kTerms; ++n) tmem_ld<H>(lanes + (i & 1) * NC + n * NH, d[n]);
          tmem_wait_ld();
#pragma unroll
          for (int g = 0; g < H; ++g) {
            u[g] = live ? fmaf(Digits<FMT>::join(d[0][g], d[1][g], d[2][g]) * ksc, s_qf[g0 + g], lv) : -INFINITY;
            m[g] = warp_max_nan(u[g]);
          }
          if (lane == 0) {
#pragma unroll
            for (int g = 0; g < H; g += 2) *reinterpret_cast<float2*>(&red_m[i & 1][quad][g0 + g]) = make_float2(m[g], m[g + 1]);
          }
        }
        named_bar(1 + wg, 128);
#pragma unroll
        for (int g = 0; g < H; g += 2) {
          float2 x[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = *reinterpret_cast<const float2*>(&red_m[i & 1][q][g0 + g]);
          m[g] = max_nan(max_nan(x[0].x, x[1].x), max_nan(x[2].x, x[3].x));
          m[g + 1] = max_nan(max_nan(x[0].y, x[1].y), max_nan(x[2].y, x[3].y));
        }
        unsigned char* Wt = Ws + (i & 1) * NC * 128;
        float l[H];
#pragma unroll
        for (int g = 0; g < H; g += 2) {
          const float w0 = ex2(u[g] - m[g]), w1 = ex2(u[g + 1] - m[g + 1]);
          l[g] = w0 * iv;
          l[g + 1] = w1 * iv;
          uint32_t dg[kTerms];
          Digits<FMT>::cut2(w0 * pow2f(Digits<FMT>::kExp), w1 * pow2f(Digits<FMT>::kExp), dg);
#pragma unroll
          for (int n = 0; n < kTerms; ++n) {
            const int c0 = n * NH + g0 + g, c1 = c0 + 1;
            Wt[c0 * 128 + (((t >> 4) ^ (c0 & 7)) * 16) + (t & 15)] = uint8_t(dg[n]);
            Wt[c1 * 128 + (((t >> 4) ^ (c1 & 7)) * 16) + (t & 15)] = uint8_t(dg[n] >> 8);
          }
        }
        const float sum = warp_sums<H>(l, lane);
        if (lane % (32 / H) == 0) red_l[i & 1][quad][g0 + lane / (32 / H)] = sum;
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(&w_full[i & 1]);
        w.next(p);
      }
      if (i > 0) {
        const int j = i - 1;
        if (j == 0 || f.c == 0) {
          s.whole = f.c == 0 && f.n <= count - j;
          s.part = f.c / f.piece;
          s.region = f.c == 0 ? blockIdx.x : s_first;
          s.clear_piece();
          s.clear_row();
        }
        wait(&o_done[j & 1], (j >> 1) & 1, kErrTimeoutMma);
        tc_fence_after();
        Fold x[H];
#pragma unroll
        for (int g = 0; g < H; g += 2) {
          float2 l[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) l[q] = *reinterpret_cast<const float2*>(&red_l[j & 1][q][g0 + g]);
          x[g] = fold_stats(s.gM[g], s.gL[g], pm[g], (l[0].x + l[1].x) + (l[2].x + l[3].x));
          x[g + 1] = fold_stats(s.gM[g + 1], s.gL[g + 1], pm[g + 1], (l[0].y + l[1].y) + (l[2].y + l[3].y));
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          uint32_t o[kTerms][H];
#pragma unroll
          for (int n = 0; n < kTerms; ++n) tmem_ld<H>(lanes + 2 * NC + ((j & 1) * KB + b) * NC + n * NH, o[n]);
          tmem_wait_ld();
#pragma unroll
          for (int g = 0; g < H; ++g)
            s.gA[b][g] = fold(s.gA[b][g], Digits<FMT>::join(o[0][g], o[1][g], o[2][g]) * pow2f(-Digits<FMT>::kExp), x[g]);
        }
        const bool last = f.c + 1 == f.n || i == count;  // of this (row, kv head) in this CTA
        // (a row's pieces of one chunk each fold like one piece: folding into an empty piece changes nothing)
        if (last || (++s.in_piece == f.piece && !(s.whole && f.piece == 1))) end_piece<H, KB>(p, f, s, g0, t, last);
        f.next(p);
      }
#pragma unroll
      for (int g = 0; g < H; ++g) pm[g] = m[g];
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_holder, kTmem);
  }
}

// Folds the (row, kv head)s that a CTA boundary cut: block (i, g) takes the one that CTA i begins inside of, if no
// earlier boundary cuts it, and query head g of its group; thread t holds head dim t. All threads fetch the pieces'
// statistics first, so that the fold, a chain of one fused multiply-add per piece, waits for one load latency per
// kMergeBatch pieces.
constexpr int kMergeBatch = 16, kMaxPieces = 512;
__global__ void __launch_bounds__(256) attn8_merge_kernel(const Args p) {
  __shared__ float2 stat[kMaxPieces];
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x + 1, g = blockIdx.y, d = threadIdx.x;
  const int4 at = p.info[i], prev = p.info[i - 1];
  const int r = at.x, h = at.y;
  if (r >= p.T || at.z == 0) return;
  if (prev.x == r && prev.y == h && prev.z > 0) return;
  const int n = at.w, ps = piece_chunks(p, n), pieces = (n + ps - 1) / ps;
  if (pieces > kMaxPieces || pieces > p.area) {
    record_error(p.err, kErrBadShape);
    return;
  }
  const int stride = p.G * (p.D + 4);
  const float* ws = p.ws + size_t(blockIdx.x) * p.area * stride + g * (p.D + 4);
  float a[kMergeBatch];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j)
      a[j] = j0 + j < pieces && d < p.D ? __ldcg(ws + size_t(j0 + j) * stride + d) : 0.f;
  };
  fetch(0);  // in flight with the statistics
  for (int j = d; j < pieces; j += blockDim.x) {
    const float* x = ws + size_t(j) * stride + p.D;
    stat[j] = make_float2(__ldcg(x), __ldcg(x + 1));
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, A = 0.f;
  for (int j0 = 0; j0 < pieces; j0 += kMergeBatch) {
    if (j0) fetch(j0);
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      if (j0 + j >= pieces) break;
      const Fold f = fold_stats(M, L, stat[j0 + j].x, stat[j0 + j].y);
      A = fold(A, a[j], f);
    }
  }
  if (d < p.D) store_out(p, r, h * p.G + g, d, A, L);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <int FMT, int NH, int KB>
void launch(Args p, int64_t bound, const torch::Tensor& q, cudaStream_t stream) {
  const int dev = q.device().index();
  auto kernel = attn8_kernel<FMT, NH, KB>;
  constexpr int smem = smem_bytes(KB, NH);
  static bool attr_set[64] = {};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set[dev] = true;
  }
  const int full = at::cuda::getCurrentDeviceProperties()->multiProcessorCount * ctas_per_sm(KB, NH);
  const int grid = int(std::min<int64_t>(bound, full));
  p.spread = full;
  // a boundary's room: all pieces of one (row, kv head)
  p.area = int(std::min<int64_t>(p.max_chunks, ceil_div(full, p.Hk)));
  const int64_t info = grid * 4;
  auto ws = torch::empty({info + int64_t(grid - 1) * p.area * p.G * (p.D + 4)}, q.options().dtype(torch::kFloat32));
  p.info = reinterpret_cast<int4*>(ws.data_ptr<float>());
  p.ws = ws.data_ptr<float>() + info;
  C10_CUDA_CHECK(launch_pdl(kernel, grid, num_threads(KB), smem, stream, p));
  if (grid > 1) C10_CUDA_CHECK(launch_pdl(attn8_merge_kernel, dim3(grid - 1, p.G), p.D <= 128 ? 128 : 256, 0, stream, p));
}

}  // namespace

// q [T, Hq, D] bf16 or fp16; codes [slots, Hk, D] float8_e4m3fn or int8, scales fp32 [Hk, slots]; returns [T, Hq * D].
// ``max_keys`` bounds every row's logical length.
torch::Tensor attention8(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& vc,
                         const torch::Tensor& ks, const torch::Tensor& vs, const torch::Tensor& bt, int64_t page,
                         const torch::Tensor& req, const torch::Tensor& start, const torch::Tensor& end,
                         const torch::Tensor& extra, const torch::Tensor& n_extra, double scale, int64_t max_keys,
                         const c10::optional<torch::Tensor>& gate) {
  const at::cuda::CUDAGuard g(q.device());
  const auto dev = q.device();
  TORCH_CHECK(q.dim() == 3 && q.is_contiguous() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
              "attention: q must be contiguous [rows, heads, head dim] in bf16 or fp16");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  const bool fp8 = kc.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(kc.dim() == 3 && kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type() &&
                  (fp8 || kc.scalar_type() == at::kChar) && kc.is_contiguous() && vc.is_contiguous() &&
                  kc.device() == dev && vc.device() == dev && kc.size(2) == D,
              "attention: 8-bit caches must be contiguous [slots, kv heads, head dim] float8_e4m3fn or int8 on q's device");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(kc.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vc.data_ptr()) % 16 == 0,
              "attention: 8-bit caches must start on a 16-byte boundary");
  const int64_t Hk = kc.size(1), slots = kc.size(0);
  for (const torch::Tensor* s : {&ks, &vs})
    TORCH_CHECK(s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == Hk && s->size(1) == slots &&
                    s->is_contiguous() && s->device() == dev,
                "attention: 8-bit caches need contiguous fp32 scales [kv heads, slots] on q's device");
  TORCH_CHECK(D % 16 == 0 && D >= 16 && D <= 256, "attention: head dim of an 8-bit cache must be a multiple of 16 up to 256");
  TORCH_CHECK(Hk > 0 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 16, "attention: query heads per kv head must be <= 16");
  TORCH_CHECK(slots * Hk < (int64_t(1) << 31), "attention: the cache has too many (slot, kv head) rows");
  TORCH_CHECK(page > 0 && page < (int64_t(1) << 31) && slots > 0 && max_keys >= 0, "attention: empty cache or page");
  TORCH_CHECK(max_keys <= (int64_t(1) << 31) - 2 * kChunk, "attention: too many keys");
  auto rows = [&](const torch::Tensor& t, const char* name, int64_t dims) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous() && t.device() == dev &&
                    (name[0] == 'b' || t.size(0) == T),
                "attention: ", name, " must be contiguous int32 with one entry per row on q's device");
    return t.data_ptr<int>();
  };
  auto out = torch::empty({T, Hq * D}, q.options());
  if (T == 0) return out;
  Args p = {};
  p.bt = rows(bt, "block_table", 2);
  p.req = rows(req, "req", 1);
  p.start = rows(start, "ctx_start", 1);
  p.end = rows(end, "ctx_len", 1);
  p.extra = rows(extra, "extra", 2);
  p.n_extra = rows(n_extra, "n_extra", 1);
  TORCH_CHECK(extra.size(1) <= kMaxExtra, "attention: at most 128 extra slots per row");
  if (gate)
    TORCH_CHECK(gate->dim() == 2 && gate->size(0) == T && gate->size(1) == Hq * D && gate->stride(1) == 1 &&
                    gate->scalar_type() == q.scalar_type() && gate->device() == dev,
                "attention: gate must be [rows, heads * head dim] in q's type");
  p.q = q.data_ptr();
  p.k = reinterpret_cast<const uint8_t*>(kc.data_ptr());
  p.v = reinterpret_cast<const uint8_t*>(vc.data_ptr());
  p.ks = ks.data_ptr<float>();
  p.vs = vs.data_ptr<float>();
  p.gate = gate ? gate->data_ptr() : nullptr;
  p.ldg = gate ? gate->stride(0) : 0;
  p.out = out.data_ptr();
  p.err = gemm_error_word(dev).data_ptr<int>();
  p.slots = slots;
  p.T = int(T);
  p.Hq = int(Hq);
  p.Hk = int(Hk);
  p.G = int(Hq / Hk);
  p.D = int(D);
  p.page = int(page);
  p.bt_ld = int(bt.size(1));
  p.bt_rows = int(bt.size(0));
  p.extra_ld = int(extra.size(1));
  p.max_chunks = int(std::max<int64_t>(1, ceil_div(max_keys, kChunk)));
  p.fp16 = q.scalar_type() == at::kHalf;
  p.scale = float(scale * 1.4426950408889634);
  const int64_t bound = T * Hk * p.max_chunks;
  TORCH_CHECK(bound < (int64_t(1) << 30), "attention: too many (row, kv head, 128-key chunk)s in one call");
  auto stream = at::cuda::getCurrentCUDAStream().stream();
#define E4_ATTN8(F, NH)                                          \
  {                                                              \
    if (D <= 128) launch<F, NH, 1>(p, bound, q, stream);         \
    else launch<F, NH, 2>(p, bound, q, stream);                  \
  }
#define E4_ATTN8_HEADS(F)                                        \
  {                                                              \
    if (p.G <= 4) E4_ATTN8(F, 4) else if (p.G <= 8) E4_ATTN8(F, 8) else E4_ATTN8(F, 16) \
  }
  if (fp8) E4_ATTN8_HEADS(kFmtFp8) else E4_ATTN8_HEADS(kFmtInt8)
  return out;
}

}  // namespace e4
