// Weight gradient of a projection whose input was kept in 8 bits:
//   out[n][k] (+)= sum over tokens m of grad[m][n] * code[m][k] * 2^e[m][k/32]
//
// A code times its power of two has seven significant bits, so it is exact in
// bfloat16 (and in float16 where the values were float16): the matrix
// instructions take gradients and kept values as they are and add in 32 bits.
// Gradients in float32 go in as three bfloat16 terms that add up to them.
//
// 16384 tokens, 8192 outputs, 8192 columns, bf16: 1.9 to 2.0 ms, 1.1 PFLOP/s (a
// library product of bf16 operands of these sizes: 1.91 ms). What bounds it is
// the issue of instructions beside the matrix instructions, which keep their
// pipes busy half of the time, and the clock, which falls with them: operands of
// zeros take 15 % less. Of 235 us for 8192 x 4096 x 4096 of those, decoding is
// 50 and the reads of LDS 14. Tried and not kept: instructions of 32 x 32 (5 %
// fewer cycles, 4 % more time); reading LDS two or three fragments ahead (no
// gain, more registers); taking the exponent off packed codes instead of two
// multiplications (a quarter fewer vector instructions, 1 % less time, and a
// second loop for exponents above 0).
// Few tiles: 2999 x 1155 x 2077 fp16 takes 45 us, of which 10 are the sums of
// five parts coming back and 6 the layout of odd rows. Small ones wait for their
// code: 56 x 208 x 355 fp32 took 28 us when stores of whole and of cut groups of
// columns stood unrolled behind the sums, and takes 14.5.
#include <hip/hip_runtime.h>
#include <type_traits>
#include "../common/act8.hpp"
#include "../common/tensor_ops.hpp"
#include "ops_device.hpp"

namespace accl {
namespace ops {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32 u32_any __attribute__((aligned(1)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A workgroup of four waves takes TN outputs by TK columns, each wave all of
// the outputs and WK columns of its own: gradients are shared through LDS,
// while codes go from memory to the registers of the one wave that needs them
// and are decoded there once. A lane holds four neighbouring columns, one in
// each of four fragments, so that it reads four codes at once, which share an
// exponent, and writes four results at once.
constexpr int TN = 128, TK = 256, WK = 64;

union Frag {
  u32 w[4];
  s16x4 h[2];
  bf16x8 b;
  f16x8 f;
};

__device__ inline f32x4 multiply(const Frag& a, const Frag& b, f32x4 c,
                                  bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
}
__device__ inline f32x4 multiply(const Frag& a, const Frag& b, f32x4 c,
                                  fp16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.f, b.f, c, 0, 0, 0);
}

// Two values as the matrix instructions take them. Both are exact, in float16
// because its exponents were bounded (scale_bits).
__device__ inline u32 pack2(float lo, float hi, bf16) {
  return __builtin_amdgcn_perm(act8::float_bits(hi), act8::float_bits(lo),
                               0x07060302);
}
__device__ inline u32 pack2(float lo, float hi, fp16) {
  auto v = __builtin_amdgcn_cvt_pkrtz(lo, hi);
  u32 w;
  __builtin_memcpy(&w, &v, 4);
  return w;
}

// 2^e as bfloat16, NaN where the group holds none (whose byte gives a number
// above all others) or one that overflows
__device__ inline u16 scale_bits(int e, u16 most) {
  const u16 scale = u16((e + 127) << 7);
  return scale > most ? u16(0x7FC0) : scale;
}
__device__ inline u16 scale_bits(int e, bf16) { return scale_bits(e, u16(0x7F00)); }
__device__ inline u16 scale_bits(int e, fp16) {
  return scale_bits(e, u16((act8::F16_MOST + 127) << 7));
}

// x as bfloat16 terms, the first ones cut short, so that they add up to x and
// none of them overflows
__device__ inline void three_terms(float x, u16 t[3]) {
  u32 b = act8::float_bits(x);
  if ((b & 0x7F800000u) == 0x7F800000u) {
    t[0] = u16(b >> 16) | ((b & 0x7FFFFFu) ? 0x40 : 0);
    t[1] = t[2] = 0;
    return;
  }
  t[0] = u16(b >> 16);
  float r = x - act8::bits_float(b & 0xFFFF0000u);
  b = act8::float_bits(r);
  t[1] = u16(b >> 16);
  r -= act8::bits_float(b & 0xFFFF0000u);
  t[2] = u16(act8::float_bits(r) >> 16);
}

// A quotient is computed in vector registers, though all lanes have the same.
__device__ inline u32 scalar(u32 v) { return __builtin_amdgcn_readfirstlane(v); }

// p, as a value that the compiler keeps in scalar registers: an address is
// then that and a lane's own 32-bit offset
template <class P>
using global = const P __attribute__((address_space(1)))*;
template <class P>
__device__ inline global<P> uniform(const P* p) {
  auto g = (global<P>)p;
  asm volatile("" : "+s"(g));
  return g;
}

// Tokens lie in LDS in groups of four: group g of a step's eight holds tokens
// g, g + 8, g + 16 and g + 24, one for each quarter of a wave. A transposing
// read takes 32 bytes of four tokens from four groups for each quarter. With 64
// bytes between groups, and neighbouring pieces of 32 bytes exchanged for every
// second quarter, two quarters meet every LDS bank once, and all reads of a lane
// are at fixed distances from two addresses.
constexpr int GROUP_STRIDE = 4 * TN + 32;

// v to (or onto) where `to` points
template <class O>
__device__ inline void put1(O* to, float v, bool add) {
  *to = O((add ? float(*to) : 0.0f) + v);
}
template <class O>
__device__ inline void put4(O* to, const float v[4], bool add) {
  struct __attribute__((packed, aligned(sizeof(O)))) Four { O e[4]; } four;
  if (add) four = *(const Four*)to;
#pragma unroll
  for (int f = 0; f < 4; ++f)
    four.e[f] = O((add ? float(four.e[f]) : 0.0f) + v[f]);
  *(Four*)to = four;
}

__device__ inline u32 here(u32 offset) {
  asm volatile("" : "+v"(offset));
  return offset;
}

// The gradients as the matrix instructions take them: 16-bit values in rows of
// a multiple of 8, at 16-byte addresses, so that they go to LDS without a stop
// in registers. Float32 gradients have three planes of them.
struct Grads {
  const u16* at;
  u32 stride, columns;
  u64 plane;
};

struct No { __device__ constexpr operator bool() const { return false; } };
struct Yes { __device__ constexpr operator bool() const { return true; } };

// E: type of the matrix instructions; DEPTH: tokens between two barriers. With
// `partial`, sums of this part of the tokens go there.
template <class E, class O, int PLANES, int DEPTH>
__global__ void __launch_bounds__(256, 2)
    weight_grad_kernel(WeightGradArgs a, Grads grads, u32 tiles_n, u32 tiles_k,
                       u32 items, u64 part_rows, float* partial) {
  constexpr int STEPS = DEPTH / 32;
  typedef u16 Buffer[PLANES][DEPTH / 4][GROUP_STRIDE];
  // two objects, so that reads of one need not wait for loads to the other
  __shared__ __align__(16) Buffer grads_even, grads_odd;
  __shared__ __align__(16) u16 scales[2][TK / 32][DEPTH];

  const u32 t = threadIdx.x, lane = t & 63;
  const u32 wave = scalar(t >> 6);
  const u32 j = lane & 15, quarter = lane >> 4;

  // neighbouring items run on one XCD and share gradients and codes in its L2
  const u32 per_xcd = gridDim.x / 8;
  const u32 item = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (item >= items) return;
  const u32 tiles = tiles_n * tiles_k, part = item / tiles, tile = item % tiles;
  const u32 band = tile / (8 * tiles_k), first = band * 8;
  const u32 high = tiles_n - first < 8 ? tiles_n - first : 8;
  const u32 in_band = tile - band * 8 * tiles_k;
  const u64 n0 = u64(scalar(first + in_band % high)) * TN;
  const u64 k0 = u64(scalar(in_band / high)) * TK;
  const u64 m_begin = scalar(part) * part_rows;  // below a.rows
  const u64 m_end = m_begin + part_rows < a.rows ? m_begin + part_rows : a.rows;

  // codes: columns k .. k + 3 of this lane. The last columns of a width that
  // is no multiple of four are read as the last ones of their four.
  const u64 k = k0 + wave * WK + 4 * j;
  const u64 k_read = k < a.width - 4 ? k : a.width - 4;
  const u32 codes_at = u32(k_read) + quarter * 8 * u32(a.codes_stride);
  const u64 group = k0 / 32 + wave * 2;  // first of this wave's two
  const u64 last_group = act8::groups_of(a.width) - 1;

  u32 fours[STEPS][8];
  int exps[DEPTH / 32];

  // ---- gradients: a wave fills a quarter of the groups, one at a time; behind
  // the last column it fetches the last eight again
  const u64 direct_n = n0 + (j ^ (2 * (quarter % 2))) * 8;
  const u32 last_n = u32((direct_n < grads.columns ? direct_n
                                                   : grads.columns - 8) - n0);
  const u32 direct_at = (quarter * 8 * grads.stride + last_n) * 2;
  auto load_grads = [&](u64 m0, Buffer& buffer) {
    const u32 row_bytes = grads.stride * 2;
#pragma unroll
    for (int q = 0; q < PLANES; ++q) {
      auto rows = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(grads.at + q * grads.plane + m0 * grads.stride + n0), 0,
          DEPTH * row_bytes, 0x00027000);
#pragma unroll
      for (int i = 0; i < DEPTH / 16; ++i) {
        const u32 g = wave * (DEPTH / 16) + i;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rows, (__attribute__((address_space(3))) void*)&buffer[q][g][0], 16,
            direct_at, (g / 8 * 32 + g % 8) * row_bytes, 0, 0);
      }
    }
  };
  // the last rows, with zeros behind them
  auto load_last_grads = [&](u64 m0, Buffer& buffer) {
    for (int q = 0; q < PLANES; ++q)
      for (u32 g = wave; g < DEPTH / 4; g += 4) {
        const u64 m = m0 + g / 8 * 32 + g % 8 + quarter * 8;
        u32x4 v = {0, 0, 0, 0};
        if (m < m_end)
          v = *(const u32x4*)(grads.at + q * grads.plane + m * grads.stride +
                              n0 + last_n);
        *(u32x4*)&buffer[q][g][lane * 8] = v;
      }
  };

  // ---- codes and exponents
  auto load_codes = [&](u64 m, int s) {
    const u32 at = here(codes_at);
#pragma unroll
    for (int r = 0; r < 8; ++r)
      fours[s][r] = *(global<u32_any>)(
          uniform(a.codes + i64(m + r) * a.codes_stride) + at);
  };
  // rows behind the last one are read from it and scaled to nothing
  auto row_of = [&](u64 m) { return i64(m < m_end ? m : m_end - 1); };
  auto load_last_codes = [&](u64 m, int s) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      fours[s][r] = *(const u32_any*)(
          a.codes + row_of(m + quarter * 8 + r) * a.codes_stride + i64(k_read));
  };
  // each wave takes the exponents of its own two groups
  constexpr int GROUPS = DEPTH / 32;  // of a lane
  auto load_exps = [&](u64 m0) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const u32 row = lane % DEPTH;
      const u64 at = group + (GROUPS == 2 ? g : lane / 32);
      exps[g] = a.exps[row_of(m0 + row) * a.exps_stride +
                       i64(at < last_group ? at : last_group)];
    }
  };
  // as bfloat16; 0 for rows behind the last
  auto store_scales = [&](u64 m0, int odd) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      scales[odd][wave * 2 + (GROUPS == 2 ? g : lane / 32)][lane % DEPTH] =
          m0 + lane % DEPTH < m_end ? scale_bits(exps[g], E()) : u16(0);
  };

  // ---- decode: rows 8 quarter .. + 7 of a step
  struct Scales { union { u32x4 q; u16 h[8]; }; };
  auto load_scales = [&](int odd, int s) {
    Scales sc;
    sc.q = *(const u32x4*)&scales[odd][wave * 2 + j / 8][s * 32 + quarter * 8];
    return sc;
  };
  auto decode = [&](const Scales& sc, int s, int p, int f) {
    return pack2(float((signed char)(fours[s][2 * p] >> (8 * f))) *
                     act8::bits_float(u32(sc.h[2 * p]) << 16),
                 float((signed char)(fours[s][2 * p + 1] >> (8 * f))) *
                     act8::bits_float(u32(sc.h[2 * p + 1]) << 16), E());
  };
  // 16 lanes read four tokens of 16 outputs and each gets one output
  auto load_outputs = [&](Buffer& buffer, int plane, int s, int i) {
    Frag g;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const u32 piece = quarter * TN + j % 4 * 4 +
                        (i % 2 ? 16 - quarter % 2 * 16 : quarter % 2 * 16);
      auto* at = &buffer[plane][s * 8 + b * 4 + j / 4][piece + i / 2 * 32];
      g.h[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)at);
    }
    return g;
  };

  f32x4 sum[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int f = 0; f < 4; ++f) sum[i][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // Sums step s of a buffer from x, and decodes step `after` with scales sc to
  // next meanwhile: one wave's vector instructions run while its matrix
  // instructions do.
  auto step = [&](Buffer& buffer, int s, const Frag(&x)[4], const Scales& sc,
                  int after, Frag(&next)[4]) {
    Frag g = load_outputs(buffer, 0, s, 0);
#pragma unroll
    for (int q = 0; q < PLANES; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        Frag ahead = g;
        if (i < 7) ahead = load_outputs(buffer, q, s, i + 1);
        else if (q + 1 < PLANES) ahead = load_outputs(buffer, q + 1, s, 0);
#pragma unroll
        for (int f = 0; f < 4; ++f)
          sum[i][f] = multiply(g, x[f], sum[i][f], E());
        g = ahead;
        if (q == 0) {
#pragma unroll
          for (int f = i % 2 * 2; f < i % 2 * 2 + 2; ++f)
            next[f].w[i / 2] = decode(sc, after, i / 2, f);
        }
      }
  };

  // Whole depths. While one is summed, the next one's gradients, and codes of
  // up to two steps ahead, are on their way; past the end the last one is
  // fetched again.
  const u32 depths = scalar(u32((m_end - m_begin) / DEPTH));
  if (depths) {
    auto row = [&](u32 d) {
      return m_begin + u64(d < depths ? d : depths - 1) * DEPTH;
    };
    Frag x[2][4];
    load_exps(m_begin);
    load_grads(m_begin, grads_even);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) load_codes(m_begin + s * 32, s);
    store_scales(m_begin, 0);
    load_exps(row(1));
    {
      const Scales sc = load_scales(0, 0);
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int f = 0; f < 4; ++f) x[0][f].w[p] = decode(sc, 0, p, f);
    }
    load_codes(row(1), 0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    auto depth = [&](u32 d, int odd, Buffer& now, Buffer& then) {
      // The scales are read before loads to LDS go out: the compiler cannot
      // tell them from what those write, and would wait for it.
      store_scales(m_begin, odd ^ 1);
      Scales sc[2];
      if constexpr (STEPS == 2) sc[0] = load_scales(odd, 1);
      sc[1] = load_scales(odd ^ 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      load_grads(row(d + 1), then);
      // loads issued from here on are later than those to LDS
      __builtin_amdgcn_sched_barrier(0);
      load_exps(row(d + 2));
      if constexpr (STEPS == 2) {
        step(now, 0, x[0], sc[0], 1, x[1]);
        load_codes(row(d + 1) + 32, 1);
        step(now, 1, x[1], sc[1], 0, x[0]);
      } else {
        step(now, 0, x[odd], sc[1], 0, x[odd ^ 1]);
      }
      load_codes(row(d + 2), 0);
      // the loads to LDS are further back than the codes of this depth's steps
      if constexpr (STEPS == 2)
        asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    for (u32 d = 0; d < depths; d += 2) {
      depth(d, 0, grads_even, grads_odd);
      if (d + 1 < depths) depth(d + 1, 1, grads_odd, grads_even);
    }
    // loads that went too far
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  }
  // what is left of the tokens
  const u64 rest = m_begin + u64(depths) * DEPTH;
  if (rest < m_end) {
    load_last_grads(rest, grads_even);
    load_exps(rest);
    store_scales(rest, 0);
    __syncthreads();
#pragma unroll 1
    for (int s = 0; s < STEPS && rest + s * 32 < m_end; ++s) {
      Frag x[4];
      load_last_codes(rest + s * 32, 0);
      const Scales sc = load_scales(0, s);
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int f = 0; f < 4; ++f) x[f].w[p] = decode(sc, 0, p, f);
#pragma unroll 1
      for (int q = 0; q < PLANES; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const Frag g = load_outputs(grads_even, q, s, i);
#pragma unroll
          for (int f = 0; f < 4; ++f)
            sum[i][f] = multiply(g, x[f], sum[i][f], E());
        }
    }
  }

  // Element e of a lane's sums is output 4 quarter + e of its fragment. Code
  // that runs once is short: fetching it is what a small product waits for.
  const u64 n_first = n0 + 4 * quarter;
  const u32 outputs =
      n_first < a.outputs
          ? u32(a.outputs - n_first < TN ? a.outputs - n_first : TN) : 0;
  auto put_tile = [&](auto* out, i64 stride, auto add) {
    if (k + 4 <= a.width) {
      auto* to = out + i64(n_first) * stride + i64(k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v[4] = {sum[i][0][e], sum[i][1][e], sum[i][2][e],
                              sum[i][3][e]};
          if (u32(i * 16 + e) < outputs) put4(to, v, add);
          to += stride;
        }
        to += 12 * stride;
      }
    }
    // the columns behind the last four, one lane's of each quarter
    const u32 behind = u32(a.width % 4);
    const u64 tail = a.width - behind;
    if (behind && tail >= k0 + wave * WK && tail < k0 + wave * WK + WK) {
      auto* shared = (float(*)[4])&grads_odd;
      if (k == tail)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int f = 0; f < 4; ++f)
              shared[i * 16 + 4 * quarter + e][f] = sum[i][f][e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (u32 at = lane; at < TN * behind; at += 64) {
        const u32 n = at / behind, f = at % behind;
        if (n0 + n >= a.outputs) break;
        auto* to = out + i64(n0 + n) * stride + i64(tail + f);
        put1(to, shared[n][4 - behind + f], add);
      }
    }
  };
  if (partial)
    put_tile(partial + u64(part) * a.outputs * a.width, i64(a.width), No());
  else if (a.accumulate)
    put_tile((O*)a.out, a.out_stride, Yes());
  else
    put_tile((O*)a.out, a.out_stride, No());
}

// Gradients of other types, rows or addresses as Grads.
template <class T, int PLANES>
__global__ void __launch_bounds__(256) lay_out_kernel(WeightGradArgs a, u16* to,
                                                      u32 columns, u64 plane) {
  const u64 c = (u64(blockIdx.x) * 64 + (threadIdx.x & 63)) * 8;
  if (c >= columns) return;
  const int n = int(a.outputs - c < 8 ? a.outputs - c : 8);
  for (u64 m = u64(blockIdx.y) * 4 + (threadIdx.x >> 6); m < a.rows;
       m += u64(gridDim.y) * 4) {
    Eight<T> v;
    load8((const T*)a.grad + i64(m) * a.grad_stride + i64(c), n, v);
    u16* row = to + m * columns + c;
    if constexpr (PLANES == 1) {
      *(u32x4*)row = v.q[0];
    } else {
      union { u16 h[3][8]; u32x4 q[3]; } t;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u16 terms[3];
        three_terms(float(v.e[e]), terms);
#pragma unroll
        for (int p = 0; p < 3; ++p) t.h[p][e] = terms[p];
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) *(u32x4*)(row + p * plane) = t.q[p];
    }
  }
}

// The parts' sums in their order, rounded once: four neighbours a thread, of one
// row or two. The gradient of 16384 x 240 x 96 bf16 took 28.6 us with a block a
// row and takes 19.4 so (23 with two parts' loads at once instead of four), that
// of 2999 x 1155 x 2077 fp16 43.9 and 44.6.
template <class O>
__global__ void __launch_bounds__(256) join_kernel(WeightGradArgs a, u32 parts,
                                                   const float* partial) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  const u64 size = a.outputs * a.width;
  for (u64 at = (u64(blockIdx.x) * 256 + threadIdx.x) * 4; at < size;
       at += u64(gridDim.x) * 1024) {
    const int n = int(size - at < 4 ? size - at : 4);
    float sums[4] = {};
    if (n == 4) {
      f32x4_any v = *(const f32x4_any*)(partial + at);
#pragma unroll 4
      for (u32 p = 1; p < parts; ++p)
        v += *(const f32x4_any*)(partial + at + p * size);
#pragma unroll
      for (int c = 0; c < 4; ++c) sums[c] = v[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < n)
          for (u32 p = 0; p < parts; ++p) sums[c] += partial[at + c + p * size];
    }
    const u64 row = size >> 32 ? at / a.width : u32(at) / u32(a.width);
    u64 k = at - row * a.width;
    O* to = (O*)a.out + i64(row) * a.out_stride + i64(k);
    if (k + 4 <= a.width) {
      put4(to, sums, a.accumulate);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c >= n) break;
        put1(to, sums[c], a.accumulate);
        if (++k < a.width) {
          ++to;
        } else {
          k = 0;
          to += a.out_stride - i64(a.width) + 1;
        }
      }
    }
  }
}

// Fewer than four columns: a block takes one column of 64 outputs, its four
// waves every fourth token each.
template <class T, class O>
__global__ void __launch_bounds__(256) column_kernel(WeightGradArgs a) {
  __shared__ float part[4][64];
  const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 n = u64(blockIdx.x) * 64 + lane;
  const i64 k = blockIdx.y;
  using In = std::conditional_t<std::is_same_v<T, fp16>, fp16, bf16>;
  float v = 0.0f;
  if (n < a.outputs)
    for (u64 m = wave; m < a.rows; m += 4)
      v += float(((const T*)a.grad)[i64(m) * a.grad_stride + i64(n)]) *
           (float(a.codes[i64(m) * a.codes_stride + k]) *
            act8::bits_float(
                u32(scale_bits(a.exps[i64(m) * a.exps_stride], In())) << 16));
  part[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && n < a.outputs) {
    O* to = (O*)a.out + i64(n) * a.out_stride + k;
    *to = O((a.accumulate ? float(*to) : 0.0f) + part[0][lane] + part[1][lane] +
            part[2][lane] + part[3][lane]);
  }
}

// Zeros, where there are no tokens.
template <class O>
__global__ void __launch_bounds__(256) nothing_kernel(WeightGradArgs a) {
  const u64 size = a.outputs * a.width;
  for (u64 i = u64(blockIdx.x) * 256 + threadIdx.x; i < size;
       i += u64(gridDim.x) * 256) {
    const u64 n = i / a.width;
    ((O*)a.out)[i64(n) * a.out_stride + i64(i - n * a.width)] = O(0.0f);
  }
}

// Tokens are split over parts where the tiles alone leave compute units idle: two
// workgroups for each of the 256 compute units (4096 x 1024 x 4096 fp32 took 108
// us, 113 with one, 121 with one and a half, 135 with four).
// A part has at least 256 tokens, or 128 that take three times the instructions
// (1600 x 750 x 71 fp32: 27.1 us with 256, 23.9 with 128; 2357 x 1721 x 99 fp16:
// 27.4 and 33.0).
// A part is a number of whole depths, so that only the last one ends inside
// one; there are no more parts than that leaves tokens for.
struct Parts {
  u64 rows;  // of a part
  u32 n;
};

static Parts parts_of(u64 rows, u64 outputs, u64 width, u64 least) {
  const u64 tiles = u64(blocks_of(outputs, TN)) * blocks_of(width, TK);
  u64 n = tiles >= 512 ? 1 : 512 / tiles;
  u64 per = (rows + n - 1) / n;
  per = per < least ? least : (per + 63) / 64 * 64;
  return {per, u32((rows + per - 1) / per)};
}

// Gradients that need not be laid out anew.
static bool as_they_are(const WeightGradArgs& a) {
  return a.dtype != DataType::float32 && a.outputs % 8 == 0 &&
         a.grad_stride % 8 == 0 && a.grad_stride < (1 << 24) &&
         u64(a.grad) % 16 == 0;
}

struct WeightGradSpace {
  u64 part_rows;
  u32 parts, columns;
  u16* grads;  // if they are laid out
  float* partial;
  u64 bytes;
  explicit WeightGradSpace(const WeightGradArgs& a) {
    const Parts p = parts_of(a.rows, a.outputs, a.width,
                             a.dtype == DataType::float32 ? 128 : 256);
    part_rows = p.rows;
    parts = p.n;
    columns = u32((a.outputs + 7) / 8 * 8);
    char* at = (char*)a.workspace;
    grads = (u16*)at;
    if (!as_they_are(a))
      at += (a.rows * columns * (a.dtype == DataType::float32 ? 6 : 2) + 255) /
            256 * 256;
    partial = parts > 1 ? (float*)at : nullptr;
    if (parts > 1) at += u64(parts) * a.outputs * a.width * sizeof(float);
    bytes = u64(at - (char*)a.workspace);
  }
};

u64 gpu_act8_weight_grad_workspace(const WeightGradArgs& a) {
  if (a.width < 4 || !a.rows || !a.outputs) return 0;
  return WeightGradSpace(a).bytes;
}

void gpu_act8_weight_grad(const WeightGradArgs& a, void* stream) {
  const char* what = "act8_weight_grad";
  if (!a.outputs || !a.width || (!a.rows && a.accumulate)) return;
  hipStream_t st = (hipStream_t)stream;
  const u64 size = a.outputs * a.width;
  const u32 flat = u32(size / 256 < 65535 ? (size + 255) / 256 : 65535);
  with_type(a.out_dtype, what, [&](auto o) {
    using O = decltype(o);
    if (!a.rows) {
      hipLaunchKernelGGL((nothing_kernel<O>), dim3(flat), dim3(256), 0, st, a);
      return;
    }
    if (a.width < 4) {
      with_type(a.dtype, what, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((column_kernel<T, O>),
                           dim3(blocks_of(a.outputs, 64), u32(a.width)),
                           dim3(256), 0, st, a);
      });
      return;
    }
    const u32 tiles_n = blocks_of(a.outputs, TN), tiles_k = blocks_of(a.width, TK);
    const WeightGradSpace w(a);
    const u64 items = u64(tiles_n) * tiles_k * w.parts;
    if (items >= (1ull << 23) || a.outputs >= (1 << 24) ||
        a.codes_stride >= (1 << 27))
      throw accl_error(std::string(what) + ": too large");
    if (a.workspace_bytes < w.bytes)
      throw accl_error(std::string(what) + ": workspace too small");
    Grads grads{(const u16*)a.grad, u32(a.grad_stride), u32(a.outputs), 0};
    if (!as_they_are(a)) {
      grads = Grads{w.grads, w.columns, w.columns, a.rows * w.columns};
      const dim3 grid(blocks_of(w.columns, 512),
                      u32(a.rows / 4 < 65535 ? (a.rows + 3) / 4 : 65535));
      if (a.dtype == DataType::float32)
        hipLaunchKernelGGL((lay_out_kernel<float, 3>), grid, dim3(256), 0, st, a,
                           w.grads, w.columns, grads.plane);
      else
        hipLaunchKernelGGL((lay_out_kernel<bf16, 1>), grid, dim3(256), 0, st, a,
                           w.grads, w.columns, grads.plane);
    }
    const u32 grid = (u32(items) + 7) / 8 * 8;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, a, grads, tiles_n,
                         tiles_k, u32(items), w.part_rows, w.partial);
    };
    switch (a.dtype) {
      case DataType::bfloat16: go(weight_grad_kernel<bf16, O, 1, 64>); break;
      case DataType::float16: go(weight_grad_kernel<fp16, O, 1, 64>); break;
      case DataType::float32: go(weight_grad_kernel<bf16, O, 3, 32>); break;
      default: throw accl_error(std::string(what) + ": type not supported");
    }
    if (w.partial)
      hipLaunchKernelGGL((join_kernel<O>),
                         dim3(u32(size / 1024 < 65535 ? (size + 1023) / 1024
                                                      : 65535)),
                         dim3(256), 0, st, a, w.parts, w.partial);
  });
  launched(what);
}

}  // namespace ops
}  // namespace accl
