// Kernels of the 8-bit key/value cache for gfx950: decode step, prompt-phase append, read-back, eviction.
//
// The cache of one layer holds K and V rows as signed bytes [B,H,L,D] with one float scale per block of T rows and head
// [B,H,L/T].  The rows of the block that is not full yet wait in fp16 in a tail [B,H,T,D]; the step that brings the last row
// of a block quantises all T of them at once, so a row is rounded to 8 bits exactly once, whatever mix of prompt pieces and
// decode steps filled its block.
//   stored row     x -> fp16, nearest-even; a non-finite value becomes 0 and a finite one stays within +-65504, so that one
//                  bad element (padding, say) can neither turn the scale of its T rows into NaN nor into infinity
//   block          scale = absmax / 127, integer = rint(x * (127 / absmax)), all in FP32; absmax = 0: zeros
// Attention reads the cache as it stands after the append: integers * scale for complete blocks, the fp16 tail behind them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_attn_kernels.hpp"
#include "prefill_attn_kernels.hpp"

#pragma clang fp contract(off)

namespace flattn {

enum { kInF32 = 0, kInF16 = 1, kInI32 = 2 }; // what q / k_new / v_new hold

struct Kv8Params {
    Params a;      // inputs, mask, positions, partials (k_cache / v_cache unused); B, H, L, scale, plan
    int8_t *k8, *v8;          // [B*H, L, D]
    float *k_scale, *v_scale; // [B*H, nblk]
    _Float16 *k_tail, *v_tail; // [B*H, T, D]
    float *weights;           // [B*H, nblk] accumulated softmax weight, or NULL
    float2 *granules;         // workspace [B*H, L / granule rows]: (reference maximum, sum of weights) of a few rows
    const int32_t *rope_rows; // [B] table rows, or NULL: a.rope_row
    int32_t table_rows;       // rows of the table, where rope_rows is given
    int32_t in_kind;
    int32_t T, t_shift;       // rows per block, log2
    int32_t nblk;             // L / T
    int32_t S;                // queries per sequence (prompt phase)
    const int32_t *tokens_per_seq; // [B] how many of them are a sequence's own, or NULL: all
    float2 *stats;            // prompt phase, workspace [B*H, S]: (maximum, sum) of every query's softmax, or NULL
    int32_t weight_queries;   // the last of them whose weights are gathered
};

// A uniform value of an input that no kernel writes while this one runs, by a scalar load.
template <typename T>
__device__ __forceinline__ T load_uniform(const T *p) { return *(const __attribute__((address_space(4))) T *)p; }

// ---------------------------------------------------------------- inputs and stored values

// N consecutive elements of an input tensor as float.  The input format is uniform: one straight run of loads each.
template <int N>
__device__ __forceinline__ void load_input(const void *base, int kind, size_t off, float inp_scale, const float *w_scale_at, float (&dst)[N])
{
    if (kind == kInF16) {
        half8 v[N / 8];
#pragma unroll
        for (int i = 0; i < N / 8; ++i) v[i] = reinterpret_cast<const half8 *>(reinterpret_cast<const _Float16 *>(base) + off)[i];
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = (float)v[i / 8][i % 8];
    } else if (kind == kInF32) {
        float4 v[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) v[i] = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + off)[i];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) { dst[4 * i] = v[i].x; dst[4 * i + 1] = v[i].y; dst[4 * i + 2] = v[i].z; dst[4 * i + 3] = v[i].w; }
    } else { // (float)acc * inp_scale * w_scale, left to right, as the other caches' kernels
        int4 v[N / 4];
        float4 w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            v[i] = reinterpret_cast<const int4 *>(reinterpret_cast<const int32_t *>(base) + off)[i];
            w[i] = reinterpret_cast<const float4 *>(w_scale_at)[i];
        }
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            dst[4 * i + 0] = __fmul_rn(__fmul_rn((float)v[i].x, inp_scale), w[i].x);
            dst[4 * i + 1] = __fmul_rn(__fmul_rn((float)v[i].y, inp_scale), w[i].y);
            dst[4 * i + 2] = __fmul_rn(__fmul_rn((float)v[i].z, inp_scale), w[i].z);
            dst[4 * i + 3] = __fmul_rn(__fmul_rn((float)v[i].w, inp_scale), w[i].w);
        }
    }
}

// The same in two steps for 16 elements, so that other loads can be issued between: raw words, then values.
struct RawInput { u32x4 w[4]; };
__device__ __forceinline__ void request_input(const void *base, int kind, size_t off, RawInput &raw)
{
    const u32x4 *src = kind == kInF16 ? reinterpret_cast<const u32x4 *>(reinterpret_cast<const _Float16 *>(base) + off)
                                      : reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint32_t *>(base) + off);
    raw.w[0] = src[0];
    raw.w[1] = src[1];
    if (kind != kInF16) {
        raw.w[2] = src[2];
        raw.w[3] = src[3];
    }
}
__device__ __forceinline__ void input_values(const RawInput &raw, int kind, float inp_scale, const float *w_scale_at, float (&dst)[16])
{
    if (kind == kInF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dst[i] = (float)__builtin_bit_cast(half8, raw.w[i / 8])[i % 8];
    } else if (kind == kInF32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dst[i] = __uint_as_float(raw.w[i / 4][i % 4]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) dst[i] = __fmul_rn(__fmul_rn((float)(int)raw.w[i / 4][i % 4], inp_scale), w_scale_at[i]);
    }
}

// RoPE of 16 consecutive elements by their table entries, from registers or from memory.
__device__ __forceinline__ void rotate_by(float (&x)[16], const float4 (&f)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float r0, r1, r2, r3;
        rope_pair(x[4 * i], x[4 * i + 1], f[i].x, f[i].y, r0, r1);
        rope_pair(x[4 * i + 2], x[4 * i + 3], f[i].z, f[i].w, r2, r3);
        x[4 * i] = r0; x[4 * i + 1] = r1; x[4 * i + 2] = r2; x[4 * i + 3] = r3;
    }
}

template <int N>
__device__ __forceinline__ void rotate_run(float (&x)[N], const float *freq_at)
{
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(freq_at + i);
        float r0, r1, r2, r3;
        rope_pair(x[i], x[i + 1], f.x, f.y, r0, r1);
        rope_pair(x[i + 2], x[i + 3], f.z, f.w, r2, r3);
        x[i] = r0; x[i + 1] = r1; x[i + 2] = r2; x[i + 3] = r3;
    }
}

__device__ __forceinline__ _Float16 stored_half(float x)
{
    const float y = fminf(fmaxf(x, -65504.f), 65504.f);
    return to_storage<_Float16>(__builtin_isfinite(x) ? y : 0.f);
}

// 127 / absmax; 0 for a block of zeros
__device__ __forceinline__ float quant_factor(float absmax) { return absmax > 0.f ? 127.0f / absmax : 0.f; }
// Four values as bytes.  |x * factor| < 127.5 by construction: no clamp.  The product is rounded to FP32, then adding 1.5 * 2^23
// rounds it to the nearest-even integer, whose low byte is the sum's low byte.
__device__ __forceinline__ uint32_t quantise4(_Float16 a, _Float16 b, _Float16 c, _Float16 d, float factor)
{
    constexpr float kShift = 12582912.0f;
    const uint32_t qa = __float_as_uint(__fmul_rn((float)a, factor) + kShift), qb = __float_as_uint(__fmul_rn((float)b, factor) + kShift);
    const uint32_t qc = __float_as_uint(__fmul_rn((float)c, factor) + kShift), qd = __float_as_uint(__fmul_rn((float)d, factor) + kShift);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(qd, qc, 0x0c0c0400u), __builtin_amdgcn_perm(qb, qa, 0x0c0c0400u), 0x05040100u);
}

template <int I>
__device__ __forceinline__ float byte_float(uint32_t x) { return (float)(int8_t)(x >> (8 * I)); }

// ---------------------------------------------------------------- reductions across the rows of a wave

__device__ __forceinline__ float swap16(float x, float &other) // other: the value of lane ^ 16 (in one of the two orders)
{
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    other = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}
__device__ __forceinline__ float swap32(float x, float &other)
{
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    other = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}

// Maximum / sum over the 64 / LPR lane groups of a wave; within a group of LPR lanes the input is the same (cross_max) or a
// value of its own per lane (cross_sum, which adds equal lanes of the groups).
template <int LPR>
__device__ __forceinline__ float cross_max(float x)
{
    float y;
    if constexpr (LPR <= 2) x = fmaxf(x, dpp_move<0x4E>(x));  // lane ^ 2
    if constexpr (LPR <= 4) x = fmaxf(x, dpp_move<0x141>(x)); // the other four of eight
    if constexpr (LPR <= 8) x = fmaxf(x, dpp_move<0x140>(x)); // the other eight of sixteen
    if constexpr (LPR <= 16) { x = swap16(x, y); x = fmaxf(x, y); }
    if constexpr (LPR <= 32) { x = swap32(x, y); x = fmaxf(x, y); }
    return x;
}
template <int LPR>
__device__ __forceinline__ float cross_sum(float x)
{
    float y;
    static_assert(LPR >= 2, "a row has at least two 16-byte chunks");
    if constexpr (LPR <= 2) x += dpp_move<0x4E>(x);                 // lane ^ 2
    if constexpr (LPR <= 4) x += __shfl_xor(x, 4);                  // (a mirror would pair unequal lanes of the groups)
    if constexpr (LPR <= 8) x += dpp_move<0x128>(x);                // row_ror:8 = lane ^ 8
    if constexpr (LPR <= 16) { x = swap16(x, y); x += y; }
    if constexpr (LPR <= 32) { x = swap32(x, y); x += y; }
    return x;
}

// Sums 16 values per lane over the lane groups and leaves a lane with a share of the sums, x[0 .. result) of elements
// 8 * (lane / 32) + 4 * (lane / 16 % 2) + i (rows of more lanes: the larger share): the first two steps exchange what the other half
// keeps, one instruction for two values, and the last ones have a quarter of the values to add.
template <int LPR>
__device__ __forceinline__ constexpr int scattered() { return LPR <= 16 ? 4 : (LPR <= 32 ? 8 : 16); }
template <int LPR>
__device__ __forceinline__ void scatter_sum(float (&x)[16])
{
    auto add = [](auto r) __attribute__((always_inline)) -> float { return __uint_as_float(r[0]) + __uint_as_float(r[1]); };
    if constexpr (LPR <= 32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = add(__builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 8]), false, false));
    }
    if constexpr (LPR <= 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = add(__builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 4]), false, false));
    }
#pragma unroll
    for (int i = 0; i < scattered<LPR>(); ++i) {
        if constexpr (LPR <= 8) x[i] += dpp_move<0x128>(x[i]); // lane ^ 8
        if constexpr (LPR <= 4) x[i] += __shfl_xor(x[i], 4);
        if constexpr (LPR <= 2) x[i] += dpp_move<0x4E>(x[i]);  // lane ^ 2
    }
}

// ---------------------------------------------------------------- decode step

template <int D>
struct Kv8Geometry {
    static constexpr int CH = D / 16;               // 16-byte chunks per row: one per lane
    static constexpr int LPR = lanes_per_row(CH);   // lanes per row
    static constexpr bool PADDED = LPR != CH;       // size_per_head 96: two of eight lanes own no chunk
    static constexpr int GPW = 64 / LPR;            // rows per wave and load instruction; at most 32, so inside one block
    static constexpr int U = 4;                     // load instructions per matrix in flight
    static constexpr int WT = GPW * U;              // rows per wave and trip
    static constexpr int GR = WT < 32 ? WT : 32;    // rows per granule of the weight sums
    static constexpr int NG = WT / GR;              // granules per trip: each has one scale
    static constexpr int BATCH = 64 / NG;           // trips whose granules fill the lanes of a wave
};

constexpr float kKv8LazyMax = 8.0f; // base-2 units: the running reference maximum may lag the true one by this much
constexpr float kQDigits = 8300000.0f; // |q| maps to at most this: three balanced base-256 digits reach 8355711
constexpr int kKv8Waves = 4;

// What thread tid needs of its first block (block tid) for the block weights: the weight so far and, where a block is at most
// four granules, those.  Requested ahead of the merge, whose loads they travel with.
template <int D>
struct FirstBlock {
    static constexpr int GR = Kv8Geometry<D>::GR, N = GR == 32 ? 4 : 0;
    float old;
    float2 g[N ? N : 1];
    template <typename LOAD>
    __device__ __forceinline__ void request(const Kv8Params &p, int bh, int P, int tid, LOAD granule)
    {
        old = 0.f;
        if (tid > P >> p.t_shift) return;
        old = p.weights[(size_t)bh * p.nblk + tid];
        const int per = p.T / GR;
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = granule(tid * per + min(i, per - 1)); // (those that nobody wrote are not used)
    }
};

// Adds the softmax weight of every block to weights[b,h,:], from the granules and the merged statistics (M, Lsum) of the
// row.  A block whose first row arrived in this step starts from 0.
template <int D, bool AHEAD, typename LOAD>
__device__ __forceinline__ void add_block_weights(const Kv8Params &p, int bh, int P, float M, float Lsum, int tid, LOAD granule, const FirstBlock<D> &first)
{
    constexpr int GR = Kv8Geometry<D>::GR;
    const int blk_new = P >> p.t_shift;
    if (!(Lsum > 0.f)) { // every key masked: the output is NaN, nothing was attended to
        if (tid == 0 && (P & (p.T - 1)) == 0) p.weights[(size_t)bh * p.nblk + blk_new] = 0.f;
        return;
    }
    const bool open = ((P + 1) & (p.T - 1)) != 0; // the last block's rows are in the tail: one granule for all of them
    const int per = p.T / GR;
    const float rl = 1.0f / Lsum;
    for (int blk = tid; blk <= blk_new; blk += kKv8Waves * 64) {
        float w = 0.f;
        const int n = open && blk == blk_new ? 1 : per;
        if (AHEAD && FirstBlock<D>::N > 0 && blk == tid) {
#pragma unroll
            for (int i = 0; i < FirstBlock<D>::N; ++i)
                if (i < n) w = fmaf(first.g[i].y, __builtin_amdgcn_exp2f(first.g[i].x - M), w);
        } else {
            for (int i = 0; i < n; ++i) {
                const float2 ms = granule(blk * per + i);
                w = fmaf(ms.y, __builtin_amdgcn_exp2f(ms.x - M), w);
            }
        }
        float *dst = p.weights + (size_t)bh * p.nblk + blk;
        const bool fresh = blk == blk_new && (P & (p.T - 1)) == 0;
        *dst = fresh ? w * rl : fmaf(w, rl, blk == tid ? first.old : *dst);
    }
}

// Granules that other workgroups, or other waves through memory, have written.
struct GranuleLoader {
    const float *at;
    __device__ __forceinline__ float2 operator()(int i) const { return make_float2(load_partial<true>(at + 2 * i), load_partial<true>(at + 2 * i + 1)); }
};
__device__ __forceinline__ GranuleLoader granule_loader(const float2 *at) { return GranuleLoader{reinterpret_cast<const float *>(at)}; }

// Merges the (m, l, o[D]) partials of the nsp splits of one (b,h), by the 256 threads of a workgroup, into a.out:
//   M = max_s m_s;  w_s = 2^(m_s - M);  out[d] = sum_s w_s o_s[d] / sum_s w_s l_s.
// D/4 threads take a split's row, 256 / (D/4) rows side by side.  Every wave forms the weights for itself, lane s that of split s,
// so that nothing but the last sum crosses waves: one memory round trip and one barrier.  COHERENT: loads that go past the
// caches which are private to a compute unit or an XCD, 16 bytes each (8 heads, 4000 rows, 33 splits: 9.3 us the step, with
// single words 9.9; with the three barriers of the other caches' merge and the weights' loads behind it 11.1; 32 heads, 1000 rows:
// 8.9 against 10.1).  Returns (M, sum of w_s l_s), in every thread.
constexpr int kLoadDeviceCoherent = 16; // cache-policy bits of the buffer builtins: bit 4 = sc1, as a device-scope atomic load has it
template <int D>
struct MergeShared {
    static constexpr int TPG = D / 4, SG = 256 / TPG; // threads per split, splits side by side (size_per_head 96: 16 threads left over)
    static constexpr int PRE = 64 / SG < 4 ? 64 / SG : 4; // rows requested with the statistics; their weights lie in one wave's lanes
    float4 acc[SG][TPG];
    float w[kCombineMaxSplits];
};
template <int D, bool COHERENT>
__device__ __forceinline__ float2 kv8_merge(const Params &a, int bh, int nsp, int tid, MergeShared<D> &sh)
{
    constexpr int TPG = MergeShared<D>::TPG, SG = MergeShared<D>::SG, PRE = MergeShared<D>::PRE, POLICY = COHERENT ? kLoadDeviceCoherent : 0;
    const int lane = tid & 63, sg = tid / TPG, t = tid % TPG;
    const bool in_group = SG * TPG == kCombineThreads || sg < SG;
    const size_t slot0 = (size_t)bh * a.split_cap;
    const __amdgpu_buffer_rsrc_t Obuf = make_buffer(a.part_o + slot0 * D), Mbuf = make_buffer(a.part_m + slot0), Lbuf = make_buffer(a.part_l + slot0);
    auto stat = [&](__amdgpu_buffer_rsrc_t buf, int s) __attribute__((always_inline)) -> float { // 0 behind the last
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buf, s < nsp ? (uint32_t)s * 4u : kLaneOutOfRange, 0u, POLICY));
    };
    auto row = [&](int s) __attribute__((always_inline)) -> float4 {
        return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(Obuf, in_group && s < nsp ? (uint32_t)(s * TPG + t) * 16u : kLaneOutOfRange, 0u, POLICY));
    };
    const float m0 = stat(Mbuf, lane), l0 = stat(Lbuf, lane);
    float4 x[PRE];
#pragma unroll
    for (int k = 0; k < PRE; ++k) x[k] = row(sg + k * SG);
    __builtin_amdgcn_sched_barrier(0);

    float M = lane < nsp ? m0 : kMaxFloor * kLog2e;
    for (int s = lane + 64; s < nsp; s += 64) M = fmaxf(M, stat(Mbuf, s));
    M = wave_max(M);
    const float w = lane < nsp ? __builtin_amdgcn_exp2f(m0 - M) : 0.f;
    float Lsum = l0 * w;
    for (int s = lane + 64; s < nsp; s += 64) Lsum = fmaf(stat(Lbuf, s), __builtin_amdgcn_exp2f(stat(Mbuf, s) - M), Lsum);
    Lsum = wave_sum(Lsum);

    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float4 y, float ws) __attribute__((always_inline)) {
        acc.x = fmaf(y.x, ws, acc.x); acc.y = fmaf(y.y, ws, acc.y); acc.z = fmaf(y.z, ws, acc.z); acc.w = fmaf(y.w, ws, acc.w);
    };
#pragma unroll
    for (int k = 0; k < PRE; ++k) add(x[k], __shfl(w, (sg + k * SG) & 63)); // (zeros behind the last)
    if (nsp > PRE * SG) { // uniform
        for (int s = tid; s < nsp; s += kCombineThreads) sh.w[s] = __builtin_amdgcn_exp2f(stat(Mbuf, s) - M);
        __syncthreads();
#pragma unroll 4
        for (int s = sg + PRE * SG; s < nsp; s += SG) add(row(s), sh.w[s]);
    }
    if (in_group) sh.acc[sg][t] = acc;
    __syncthreads();
    if (tid < TPG) {
        float4 r = sh.acc[0][tid];
#pragma unroll
        for (int k = 1; k < SG; ++k) {
            const float4 y = sh.acc[k][tid];
            r.x += y.x; r.y += y.y; r.z += y.z; r.w += y.w;
        }
        reinterpret_cast<float4 *>(a.out + (size_t)bh * D)[tid] = make_float4(r.x / Lsum, r.y / Lsum, r.z / Lsum, r.w / Lsum);
    }
    return make_float2(M, Lsum);
}

// Quantises one full tail (T rows of one (b,h)) into block `blk`, by the 256 threads of a workgroup.  Two passes over
// the tail: T * D halfs, which the second finds in the caches.
template <int D>
__device__ __forceinline__ void quantise_tail(const _Float16 *tail, int8_t *rows8, float *scale_at, int T, float *s_red)
{
    const int tid = threadIdx.x, n8 = T * (D / 8);
    const half8 *src = reinterpret_cast<const half8 *>(tail);
    float absmax = 0.f;
    for (int i = tid; i < n8; i += kKv8Waves * 64) {
        const half8 x = src[i];
#pragma unroll
        for (int j = 0; j < 8; ++j) absmax = fmaxf(absmax, fabsf((float)x[j]));
    }
    absmax = wave_max(absmax);
    __syncthreads(); // s_red is free
    if ((tid & 63) == 0) s_red[tid >> 6] = absmax;
    __syncthreads();
    absmax = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float f = quant_factor(absmax);
    for (int i = tid; i < n8; i += kKv8Waves * 64) {
        const half8 x = src[i];
        uint2 o;
        o.x = quantise4(x[0], x[1], x[2], x[3], f);
        o.y = quantise4(x[4], x[5], x[6], x[7], f);
        reinterpret_cast<uint2 *>(rows8)[i] = o;
    }
    if (tid == 0) *scale_at = absmax / 127.0f;
}

// Whether sequence b's device-side position lies in the cache and the plan, and its table row in the table.
__device__ __forceinline__ bool kv8_position_ok(const Kv8Params &p, int b, int P)
{
    if (P < 0 || P >= p.a.L || P > p.a.max_pos) return false;
    return !p.rope_rows || (uint32_t)load_uniform(p.rope_rows + b) < (uint32_t)p.table_rows;
}

// Tokens that sequence b brings to a prompt of S; -1 where its entry lies outside [0, S].
__device__ __forceinline__ int kv8_prompt_tokens(const Kv8Params &p, int b)
{
    const int n = p.tokens_per_seq ? load_uniform(p.tokens_per_seq + b) : p.S;
    return (uint32_t)n <= (uint32_t)p.S ? n : -1;
}
// What a query behind a sequence's tokens gets: zeros, or NaN where their number is unusable.
__device__ __forceinline__ float kv8_no_query(int tokens) { return tokens < 0 ? __builtin_nanf("") : 0.f; }

// Splits of one (b,h) in a decode step whose context is split: `chunk` rows of the complete blocks each, and one more for the
// newest row and the open block's rows before it (or for the block that the newest row completes).
__device__ __forceinline__ int kv8_splits(const Params &a, int T, int P) { return (P - (P & (T - 1)) + a.chunk - 1) / a.chunk + 1; }

// One decode step (PROMPT = false): grid = splits * B * H workgroups of four waves, (b,h) fastest as in the streaming
// kernel of the other cache types.  PROMPT = true: one workgroup per (b, query, h) over the rows as they are, no append — the
// prompt phase of the head sizes the matrix-core kernel does not serve.
//
// A row of D bytes is D/16 lanes; a wave takes four load instructions of K and four of V per trip.  Scores: the query enters
// as integers of three base-256 digits, q = qs * (d0 + 256 d1 + 65536 d2) with |error| <= 2^-24 of its largest element, so K
// needs no conversion: twelve v_dot4_i32_i8 per 16 bytes multiply the bytes as they come (exactly), against 32 instructions
// for conversion and FMA.  V bytes are converted (one instruction each) and accumulated in FP32.  The running maximum is
// shared by the whole wave, which makes the weights of different rows comparable at once (granule sums) and the rescale of
// the accumulators a rare, wave-uniform branch.
//
// Bound by HBM at large batches: the loads never stop.  K of the next trip is requested into K's registers as soon as the
// scores are formed, V's as soon as V is used up, so either half of a trip's arithmetic has the other matrix's loads in
// flight, at no register's cost; the first trip is requested before the query has arrived.  B=64, 32 heads, D = 128, 2041
// rows, mask and weights: 169 us for 1.104 GB (counted: 1.103), 6.5 TB/s of the 7.1 that two streams of plain reads reach;
// without any arithmetic the same loads take as long.  Three waves per SIMD: a fourth (128 registers) changes nothing where
// it does not spill, and costs a quarter of the time where it does.  One long sequence (32 heads, 4083 rows, 9 splits): 12 us, 7
// behind the streaming and before it.
template <int D, bool HAS_MASK, bool PROMPT>
__global__ __launch_bounds__(kKv8Waves * 64) __attribute__((amdgpu_waves_per_eu(D > 512 ? 2 : 3, 8)))
void kv8_attn_kernel(const Kv8Params p)
{
    typedef Kv8Geometry<D> G;
    constexpr int LPR = G::LPR, GPW = G::GPW, U = G::U, WT = G::WT, GR = G::GR;
    constexpr bool CHECK = WT > 32; // a trip may reach over the end of the rows (blocks are multiples of 32)
    static_assert(kKv8Waves * 64 == kCombineThreads, "the merge runs on a 256-thread workgroup");
    __shared__ __attribute__((aligned(16))) float s_o[kKv8Waves][D];
    __shared__ float s_m[kKv8Waves], s_l[kKv8Waves], s_t[kKv8Waves], s_red[kKv8Waves];
    __shared__ __attribute__((aligned(16))) char s_merge_bytes[PROMPT ? 16 : sizeof(MergeShared<D>)];
    constexpr int LDS_GRANULES = (int)sizeof(s_merge_bytes) / 8; // where one workgroup has all rows and does not merge
    __shared__ int s_last;

    const Params &a = p.a;
    // One argument of every 64-byte line at once: fetched where they are first used, the lines cost three more scalar round trips
    // before the first request (0.1-0.2 us).
    asm volatile("" ::"s"(a.q), "s"(p.k8), "s"(p.in_kind), "s"(p.T));
    const int H = a.H, L = a.L, T = p.T;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane / LPR, lig = lane % LPR;
    int split = 0, bh, b, h, P, s_query = 0;
    if constexpr (PROMPT) { // blockIdx = (b * S + s) * H + h
        h = blockIdx.x % H;
        const int bs = blockIdx.x / H;
        b = bs / p.S;
        s_query = bs % p.S;
        bh = b * H + h;
        const int tokens = kv8_prompt_tokens(p, b);
        if (s_query >= tokens) {
            for (int d = tid; d < D; d += kKv8Waves * 64) a.out[((size_t)bh * p.S + s_query) * D + d] = kv8_no_query(tokens);
            return;
        }
        P = a.start_pos + tokens - 1; // the last row in the cache
    } else {
        const int BH = a.B * H;
        split = blockIdx.x / BH;
        bh = blockIdx.x % BH;
        b = bh / H;
        h = bh % H;
        P = a.pos_per_seq ? load_uniform(a.pos_per_seq + b) : a.start_pos;
        if (!kv8_position_ok(p, b, P)) { // store nothing, poison the output
            if ((a.direct || a.arrivals) && split == 0)
                for (int d = tid; d < D; d += kKv8Waves * 64) a.out[(size_t)bh * D + d] = __builtin_nanf("");
            return;
        }
    }
    const bool direct = PROMPT || a.direct;
    const int ctx = P + 1, P0 = P & ~(T - 1);
    const bool fills = ctx == P0 + T;                  // the newest row is the last of its block
    const int splits = direct ? 1 : kv8_splits(a, T, P);
    if (split >= splits) return;
    const bool owner = split == splits - 1;            // this workgroup has the newest row and the open block
    const int start = direct ? 0 : (owner ? P0 : split * a.chunk);
    const int end8 = owner ? (fills ? ctx : P0) : min(start + a.chunk, P0); // rows [start, end8) come as bytes: whole blocks
    const int q_pos = PROMPT ? a.start_pos + s_query : P;
    const size_t row_off = (size_t)bh * L * D, tail_off = (size_t)bh * T * D;
    const bool has_chunk = !G::PADDED || lig < G::CH;
    const int e0 = lig * 16, e0_in = has_chunk ? e0 : 0; // (lanes without a chunk load the first one and drop it)

    const int kind = p.in_kind;
    const float inp_scale = kind == kInI32 ? load_uniform(a.inp_scale + (PROMPT ? b * p.S + s_query : b)) : 0.f;
    int rope_row = PROMPT ? (a.rope_row < 0 ? q_pos : a.rope_row + s_query) : (a.rope_row < 0 ? P : a.rope_row);
    if (!PROMPT && p.rope_rows) rope_row = load_uniform(p.rope_rows + b);
    const float *freq = a.freq_cis + (size_t)rope_row * D + e0_in;
    const size_t in_off = PROMPT ? ((size_t)(b * p.S + s_query) * H + h) * D + e0_in : (size_t)bh * D + e0_in;

    // What a trip needs, in two halves.  A lane behind the last row reads nothing and receives zeros.
    const __amdgpu_buffer_rsrc_t Kbuf = make_buffer(p.k8 + row_off), Vbuf = make_buffer(p.v8 + row_off);
    const float *mrow = HAS_MASK ? a.attn_mask + (size_t)q_pos * a.mask_ld : nullptr;
    const __amdgpu_buffer_rsrc_t Mbuf = make_buffer(HAS_MASK ? (const void *)mrow : (const void *)p.k8);
    const float *ks_at = p.k_scale + (size_t)bh * p.nblk, *vs_at = p.v_scale + (size_t)bh * p.nblk;
    const uint32_t lane_off = has_chunk ? (uint32_t)(g * D + e0) : kLaneOutOfRange;
    u32x4 kv[U], vv[U];
    // Mask entries: a lane fetches that of row u = lane % 4 of its group, and a quad broadcast hands entry u to every lane (one
    // load and one register for the trip); rows of two lanes fetch one by one.
    constexpr bool MASK_QUAD = LPR >= 4;
    float mk[MASK_QUAD ? 1 : U];
    const uint32_t mask_lane = (uint32_t)((MASK_QUAD ? (lane & 3) * GPW : 0) + g);
    auto request_k = [&](int r) __attribute__((always_inline)) {
        if constexpr (HAS_MASK) {
#pragma unroll
            for (int u = 0; u < (MASK_QUAD ? 1 : U); ++u) {
                const bool in = r + u * GPW + (int)mask_lane < end8;
                mk[u] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(Mbuf, in ? mask_lane * 4u : kLaneOutOfRange, (uint32_t)(r + u * GPW) * 4u, 0));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = r + (CHECK ? u * GPW : 0) < end8; // uniform
            kv[u] = __builtin_amdgcn_raw_buffer_load_b128(Kbuf, in ? lane_off : kLaneOutOfRange, (uint32_t)(r + u * GPW) * (uint32_t)D, kLoadNonTemporal);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto request_v = [&](int r) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = r + (CHECK ? u * GPW : 0) < end8;
            vv[u] = __builtin_amdgcn_raw_buffer_load_b128(Vbuf, in ? lane_off : kLaneOutOfRange, (uint32_t)(r + u * GPW) * (uint32_t)D, kLoadNonTemporal);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    int r = start + wave * WT;
    // Scales: lane i holds those of granule i of the next BATCH trips, one load for all of them, and the trip that needs them
    // reads that lane.  (A block that was never written may have any scale: rows behind the last take 0.)
    float ks_lanes, vs_lanes;
    auto lane_row = [&](int base) __attribute__((always_inline)) -> int { return base + lane / G::NG * (kKv8Waves * WT) + lane % G::NG * GR; };
    auto request_scales = [&](int base) __attribute__((always_inline)) {
        const int row = lane_row(base), blk = min(row >> p.t_shift, p.nblk - 1);
        ks_lanes = row < end8 ? ks_at[blk] : 0.f;
        vs_lanes = row < end8 ? vs_at[blk] : 0.f;
    };

    // Everything whose address is known is requested before anything is waited for: the query, the new row, the first two tail
    // rows of every lane group, then the first trip of the byte rows.
    const bool appends = !PROMPT && owner, has_tail = owner && !fills;
    const bool gather = !PROMPT && p.weights != nullptr;
    RawInput q_raw, k_raw, v_raw;
    request_input(a.q, kind, in_off, q_raw);
    float4 fr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) fr[i] = reinterpret_cast<const float4 *>(freq)[i];
    if (appends && wave == 0) {
        request_input(a.k_new, kind, in_off, k_raw);
        request_input(a.v_new, kind, in_off, v_raw);
    }
    constexpr int UT = 2; // tail rows per lane group and trip
    const int n_tail = PROMPT ? ctx - P0 : P - P0; // rows to be read: the newest comes from registers
    half8 kx[UT][2], vx[UT][2];
    float mt[UT];
    auto request_tail = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UT; ++u) {
            const int at = min(r0 + u * GPW + g, n_tail - 1);
            const half8 *kt = reinterpret_cast<const half8 *>(p.k_tail + tail_off + e0_in + (size_t)at * D);
            const half8 *vt = reinterpret_cast<const half8 *>(p.v_tail + tail_off + e0_in + (size_t)at * D);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                kx[u][c] = __builtin_nontemporal_load(kt + c);
                vx[u][c] = __builtin_nontemporal_load(vt + c);
            }
            mt[u] = HAS_MASK ? mrow[P0 + at] : 0.f;
        }
    };
    if (has_tail && wave * GPW * UT < n_tail) request_tail(wave * GPW * UT);
    float mask_new = 0.f;
    if (HAS_MASK && appends) mask_new = mrow[P] * kLog2e;
    FirstBlock<D> first_block;
    if (gather && direct && tid <= P >> p.t_shift) first_block.old = p.weights[(size_t)bh * p.nblk + tid];
    __builtin_amdgcn_sched_barrier(0);
    if (!(appends && fills)) {
        request_scales(r);
        request_k(r);
        request_v(r);
    }

    // The append: the new row goes to the tail; where it completes the block, the workgroup quantises the tail, and
    // the loop below finds those rows as bytes.
    half8 kn[2], vn[2];
    if (appends) {
        if (wave == 0) {
            float x[16], y[16];
            input_values(k_raw, kind, inp_scale, kind == kInI32 ? a.wk_scale + h * D + e0_in : nullptr, x);
            input_values(v_raw, kind, inp_scale, kind == kInI32 ? a.wv_scale + h * D + e0_in : nullptr, y);
            rotate_by(x, fr);
#pragma unroll
            for (int i = 0; i < 16; ++i) { kn[i / 8][i % 8] = stored_half(x[i]); vn[i / 8][i % 8] = stored_half(y[i]); }
            if (g == 0 && has_chunk) {
                const size_t at = tail_off + (size_t)(P - P0) * D + e0;
                half8 *kd = reinterpret_cast<half8 *>(p.k_tail + at), *vd = reinterpret_cast<half8 *>(p.v_tail + at);
                kd[0] = kn[0]; kd[1] = kn[1];
                vd[0] = vn[0]; vd[1] = vn[1];
            }
        }
        if (fills) {
            __syncthreads(); // the new row is in the tail
            const int blk = P >> p.t_shift;
            quantise_tail<D>(p.k_tail + tail_off, p.k8 + row_off + (size_t)P0 * D, p.k_scale + (size_t)bh * p.nblk + blk, T, s_red);
            quantise_tail<D>(p.v_tail + tail_off, p.v8 + row_off + (size_t)P0 * D, p.v_scale + (size_t)bh * p.nblk + blk, T, s_red);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads(); // and the block in the cache
            request_scales(r);
            request_k(r);
            request_v(r);
        }
    }

    // The rotated query
    float qf[16];
    input_values(q_raw, kind, inp_scale, kind == kInI32 ? a.wq_scale + h * D + e0_in : nullptr, qf);
    rotate_by(qf, fr);
#pragma unroll
    for (int i = 0; i < 16; ++i) qf[i] = has_chunk ? qf[i] : 0.f;

    const float scale = a.scale * kLog2e;
    float m = kMaxFloor * kLog2e, l = 0.f, lt = 0.f; // wave-uniform maximum; this lane group's sums over all rows / the tail rows
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    auto raise = [&](float top) __attribute__((always_inline)) { // top: wave-uniform
        if (__builtin_amdgcn_readfirstlane((int)(top > m + kKv8LazyMax))) {
            const float alpha = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= alpha;
            lt *= alpha;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= alpha;
        }
    };

    // The tail: fp16 rows [P0, P], the newest from registers.
    if (has_tail) {
        for (int r0 = wave * GPW * UT; r0 < n_tail; r0 += kKv8Waves * GPW * UT) {
            if (r0 >= kKv8Waves * GPW * UT) request_tail(r0);
            float s[UT];
#pragma unroll
            for (int u = 0; u < UT; ++u) {
                float acc = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc = fmaf((float)kx[u][i / 8][i % 8], qf[i], acc);
                s[u] = acc;
            }
            group_sum_n<LPR, UT>(s);
            float top = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < UT; ++u) {
                s[u] = HAS_MASK ? fmaf(s[u], scale, mt[u] * kLog2e) : s[u] * scale;
                if (r0 + u * GPW + g >= n_tail) s[u] = -__builtin_inff();
                top = fmaxf(top, s[u]);
            }
            raise(cross_max<LPR>(top));
#pragma unroll
            for (int u = 0; u < UT; ++u) {
                const float e = __builtin_amdgcn_exp2f(s[u] - m);
                l += e;
                lt += e;
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = fmaf(e, (float)vx[u][i / 8][i % 8], o[i]);
            }
        }
        if (!PROMPT && wave == 0) { // the new row: every lane group has it, group 0 counts it
            float acc = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc = fmaf((float)kn[i / 8][i % 8], qf[i], acc);
            acc = group_sum<LPR>(acc);
            const float s = HAS_MASK ? fmaf(acc, scale, mask_new) : acc * scale;
            raise(s);
            if (g == 0) {
                const float e = __builtin_amdgcn_exp2f(s - m);
                l += e;
                lt += e;
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = fmaf(e, (float)vn[i / 8][i % 8], o[i]);
            }
        }
    }

    // The query as three digits per element, to 2^-24 of the head's largest one: a score is off by that much of max|q| sum|k|, as
    // sums in FP32 are.  A non-finite element makes the factor NaN, as it would every score.
    uint32_t qd[3][4];
    float qs;
    {
        float top = 0.f, bad = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { top = fmaxf(top, fabsf(qf[i])); bad += qf[i] * 0.f; }
        if constexpr (LPR >= 2) top = fmaxf(top, dpp_move<0xB1>(top));
        if constexpr (LPR >= 4) top = fmaxf(top, dpp_move<0x4E>(top));
        if constexpr (LPR >= 8) top = fmaxf(top, dpp_move<0x141>(top));
        if constexpr (LPR >= 16) top = fmaxf(top, dpp_move<0x140>(top));
        if constexpr (LPR >= 32) top = fmaxf(top, __shfl_xor(top, 16));
        if constexpr (LPR >= 64) top = fmaxf(top, __shfl_xor(top, 32));
        bad = group_sum<LPR>(bad);
        top = fmaxf(top, 1e-30f);
        const float f = kQDigits / top;
        qs = (top / kQDigits + bad) * scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = (uint32_t)((int)rintf(qf[4 * j + i] * f) + 0x808080); // digits + 128, in bytes
#pragma unroll
            for (int d = 0; d < 3; ++d)
                qd[d][j] = (((y[0] >> (8 * d)) & 0xffu) | ((y[1] >> (8 * d)) & 0xffu) << 8 | ((y[2] >> (8 * d)) & 0xffu) << 16 |
                            ((y[3] >> (8 * d)) & 0xffu) << 24) ^ 0x80808080u;
        }
    }

    // The byte rows
    float gran_m = 0.f, gran_s = 0.f; // lane i: granule i of the current batch
    float2 *const gran_at = gather ? p.granules + (size_t)bh * (L / GR) : nullptr;
    float2 *const gran_lds = reinterpret_cast<float2 *>(s_merge_bytes);
    const bool gran_local = direct && ctx <= LDS_GRANULES * GR;
    int trip = 0, batch_row = r;
    auto flush_granules = [&]() __attribute__((always_inline)) {
        const int row = lane_row(batch_row);
        if (row < min(r, end8)) { // of the trips that have been made (r: the next one)
            if (gran_local) {
                gran_lds[row / GR] = make_float2(gran_m, gran_s);
            } else {
                float *dst = reinterpret_cast<float *>(gran_at + row / GR);
                store_partial<true>(dst, gran_m);
                store_partial<true>(dst + 1, gran_s);
            }
        }
    };
    while (r < end8) {
        const int next = r + kKv8Waves * WT;
        float s[U], ks[G::NG], vs[G::NG];
#pragma unroll
        for (int n = 0; n < G::NG; ++n) {
            ks[n] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_lanes), trip * G::NG + n));
            vs[n] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_lanes), trip * G::NG + n));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int acc[3] = {0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int d = 0; d < 3; ++d) acc[d] = __builtin_amdgcn_sdot4((int)kv[u][j], (int)qd[d][j], acc[d], false);
            // 16 products of at most 127 * 128: the two low digits fit one integer, the top digit's weight is 65536
            s[u] = fmaf((float)acc[2], 65536.f, (float)(acc[0] + (acc[1] << 8)));
        }
        group_sum_n<LPR, U>(s);
        float mu[U];
        if constexpr (HAS_MASK) {
            if constexpr (MASK_QUAD) {
                const float mq = mk[0] * kLog2e;
                mu[0] = dpp_move<0x00>(mq); mu[1] = dpp_move<0x55>(mq); mu[2] = dpp_move<0xAA>(mq); mu[3] = dpp_move<0xFF>(mq);
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) mu[u] = mk[MASK_QUAD ? 0 : u] * kLog2e;
            }
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float f = qs * ks[u * GPW / GR];
            s[u] = HAS_MASK ? fmaf(s[u], f, mu[u]) : s[u] * f;
            if (CHECK && r + u * GPW >= end8) s[u] = -__builtin_inff();
            top = fmaxf(top, s[u]);
        }
        __builtin_amdgcn_sched_barrier(0);
        request_k(next); // (nothing is read behind the last row)
        raise(cross_max<LPR>(top));
        float e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            e[u] = __builtin_amdgcn_exp2f(s[u] - m);
            l += e[u];
        }
        if (gather) {
            constexpr int UG = U / G::NG; // load instructions per granule
#pragma unroll
            for (int n = 0; n < G::NG; ++n) { // (a granule is whole or absent: blocks are multiples of it)
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < UG; ++u) sum += e[n * UG + u];
                sum = cross_sum<LPR>(sum);
                const bool mine = lane == trip * G::NG + n;
                gran_m = mine ? m : gran_m;
                gran_s = mine ? sum : gran_s;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = e[u] * vs[u * GPW / GR];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[4 * j + 0] = fmaf(w, byte_float<0>(vv[u][j]), o[4 * j + 0]);
                o[4 * j + 1] = fmaf(w, byte_float<1>(vv[u][j]), o[4 * j + 1]);
                o[4 * j + 2] = fmaf(w, byte_float<2>(vv[u][j]), o[4 * j + 2]);
                o[4 * j + 3] = fmaf(w, byte_float<3>(vv[u][j]), o[4 * j + 3]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        request_v(next);
        r = next;
        if (++trip == G::BATCH) { // (uniform)
            if (gather) flush_granules();
            trip = 0;
            batch_row = r;
            request_scales(r);
        }
    }
    if (gather) flush_granules();

    // Merge: lane groups in registers, waves through LDS.
    scatter_sum<LPR>(o);
    l = cross_sum<LPR>(l);
    lt = cross_sum<LPR>(lt);
    if ((LPR > 16 || (lane & 15) < LPR) && has_chunk) {
        const int at = e0 + (LPR <= 32 ? 8 * (lane >> 5) : 0) + (LPR <= 16 ? 4 * (lane >> 4 & 1) : 0);
#pragma unroll
        for (int i = 0; i < scattered<LPR>(); i += 4) *reinterpret_cast<float4 *>(&s_o[wave][at + i]) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
        s_t[wave] = lt;
    }
    __syncthreads();
    float M = s_m[0];
#pragma unroll
    for (int w = 1; w < kKv8Waves; ++w) M = fmaxf(M, s_m[w]);
    float f[kKv8Waves], Lsum = 0.f, Lt = 0.f;
#pragma unroll
    for (int w = 0; w < kKv8Waves; ++w) {
        f[w] = __builtin_amdgcn_exp2f(s_m[w] - M);
        Lsum = fmaf(s_l[w], f[w], Lsum);
        Lt = fmaf(s_t[w], f[w], Lt);
    }
    if (gather && has_tail && tid == 0) { // the open block's weight as its first granule
        if (gran_local) {
            gran_lds[P0 / GR] = make_float2(M, Lt);
        } else {
            float *dst = reinterpret_cast<float *>(gran_at + P0 / GR);
            store_partial<true>(dst, M);
            store_partial<true>(dst + 1, Lt);
        }
    }
    const size_t slot = (size_t)bh * a.split_cap + split;
    for (int d = tid; d < D; d += kKv8Waves * 64) {
        float O = 0.f;
#pragma unroll
        for (int w = 0; w < kKv8Waves; ++w) O = fmaf(s_o[w][d], f[w], O);
        if (direct) a.out[(PROMPT ? (size_t)bh * p.S + s_query : (size_t)bh) * D + d] = O / Lsum;
        else store_partial<true>(a.part_o + slot * D + d, O);
    }
    if constexpr (!PROMPT) {
        if (direct) {
            if (gather) {
                if (!gran_local) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads(); // every wave's granules are written
                if (gran_local) add_block_weights<D, false>(p, bh, P, M, Lsum, tid, [&](int i) __attribute__((always_inline)) { return gran_lds[i]; }, first_block);
                else add_block_weights<D, false>(p, bh, P, M, Lsum, tid, granule_loader(gran_at), first_block);
            }
            return;
        }
        if (tid == 0) {
            store_partial<true>(a.part_m + slot, M);
            store_partial<true>(a.part_l + slot, Lsum);
        }
        if (!a.arrivals) return;
        // Publish -> count -> merge, ordered as in the streaming kernel of the other cache types: device-coherent stores, a
        // wait for their acknowledgement in every thread, the barrier, the device-scope count, the barrier, device-coherent
        // loads.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const int before = __hip_atomic_fetch_add(a.arrivals + bh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = before == splits - 1;
            if (before == splits - 1) __hip_atomic_store(a.arrivals + bh, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (s_last) {
            if (gather) first_block.request(p, bh, P, tid, granule_loader(gran_at));
            const float2 ml = kv8_merge<D, true>(a, bh, splits, tid, *reinterpret_cast<MergeShared<D> *>(s_merge_bytes));
            if (gather) add_block_weights<D, true>(p, bh, P, ml.x, ml.y, tid, granule_loader(gran_at), first_block);
        }
    }
}

// grid = B*H, block = 256: the merge as a launch of its own.
template <int D>
__global__ __launch_bounds__(kCombineThreads) void kv8_combine_kernel(const Kv8Params p)
{
    __shared__ MergeShared<D> sh;
    const int bh = blockIdx.x, tid = threadIdx.x, b = bh / p.a.H;
    const int P = p.a.pos_per_seq ? p.a.pos_per_seq[b] : p.a.start_pos;
    if (!kv8_position_ok(p, b, P)) {
        for (int d = tid; d < D; d += kCombineThreads) p.a.out[(size_t)bh * D + d] = __builtin_nanf("");
        return;
    }
    const GranuleLoader granule = granule_loader(p.granules + (size_t)bh * (p.a.L / Kv8Geometry<D>::GR));
    FirstBlock<D> first;
    if (p.weights) first.request(p, bh, P, tid, granule);
    const float2 ml = kv8_merge<D, false>(p.a, bh, kv8_splits(p.a, p.T, P), tid, sh);
    if (p.weights) add_block_weights<D, true>(p, bh, P, ml.x, ml.y, tid, granule, first);
}

// ---------------------------------------------------------------- prompt phase: append

// grid = max(complete blocks, 1) * 2 * B*H: one workgroup per block of rows that the call completes, K and V apart, heads
// fastest (neighbours read neighbouring heads of the same tokens); block = 256.  The first workgroup of a (b,h) is the one that reads the tail (its block may begin with rows of an
// earlier call), and therefore also the one that stores the rows of the last, incomplete block there, behind a barrier.
// Bound by the traffic: inputs once, a byte per value out.  B=8, S=1024, 32 heads, fp16: 43 us for 201 MB (4.7 TB/s; one
// chunk at a time behind a branch 56, plain instead of non-temporal loads 52; two chunks at a time or eight waves per SIMD: the
// same 43).
template <int D, int T>
__global__ __launch_bounds__(256) void kv8_append_kernel(const Kv8Params p)
{
    constexpr int CPR = D / 8;                        // 8-element chunks per row
    constexpr int NI = (T * CPR + 255) / 256;         // chunks per thread
    constexpr bool EXACT = (T * CPR) % 256 == 0;
    constexpr bool KEEP = NI <= 16;                   // the rounded rows stay in registers between the two passes
    __shared__ float s_red[4];
    const Params &a = p.a;
    const int BH = a.B * a.H;
    const int tid = threadIdx.x, bh = blockIdx.x % BH, b = bh / a.H, h = bh % a.H;
    const bool is_v = (blockIdx.x / BH & 1) != 0;
    const int nth = blockIdx.x / BH >> 1; // of the blocks this call touches
    const int P = a.start_pos, end = P + max(kv8_prompt_tokens(p, b), 0);
    const int first = P / T, last = end / T;          // blocks [first, last) are complete after the call
    _Float16 *tail = (is_v ? p.v_tail : p.k_tail) + (size_t)bh * T * D;
    const void *src = is_v ? a.v_new : a.k_new;
    const float *w = is_v ? a.wv_scale : a.wk_scale;

    auto new_chunk = [&](int row, int e0) __attribute__((always_inline)) -> half8 { // row of the cache, P <= row < end
        const int64_t token = (int64_t)b * p.S + (row - P);
        const float inp_scale = p.in_kind == kInI32 ? a.inp_scale[token] : 0.f;
        float x[8];
        load_input<8>(src, p.in_kind, (size_t)(token * a.H + h) * D + e0, inp_scale, p.in_kind == kInI32 ? w + h * D + e0 : nullptr, x);
        if (!is_v) rotate_run<8>(x, a.freq_cis + (size_t)(a.rope_row < 0 ? row : a.rope_row + (row - P)) * D + e0);
        half8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = stored_half(x[i]);
        return y;
    };
    const int blk = first + nth;
    if (blk < last) {
        auto chunk = [&](int i) __attribute__((always_inline)) -> half8 { // chunk i of the block's T * CPR
            const int row = blk * T + i / CPR, e0 = (i % CPR) * 8;
            if (row < P) return *reinterpret_cast<const half8 *>(tail + (size_t)(i / CPR) * D + e0);
            return new_chunk(row, e0);
        };
        half8 kept[KEEP ? NI : 1];
        float absmax = 0.f;
        if (KEEP && blk * T >= P) {
            // every row is new: the loads of a batch of chunks are issued before the first value is used
            auto load_block = [&](auto kind_tag, auto v_tag) __attribute__((always_inline)) {
                constexpr int KIND = decltype(kind_tag)::value, BATCH = NI < 4 ? NI : 4;
                constexpr bool IS_V = decltype(v_tag)::value != 0;
#pragma unroll
                for (int n0 = 0; n0 < NI; n0 += BATCH) {
                    u32x4 raw[BATCH][KIND == kInF16 ? 1 : 2];
                    float4 fr[BATCH][IS_V ? 1 : 2], ws[KIND == kInI32 ? BATCH : 1][2];
                    float sc[KIND == kInI32 ? BATCH : 1];
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) {
                        if (n0 + j >= NI) continue;
                        const int i = EXACT ? tid + (n0 + j) * 256 : min(tid + (n0 + j) * 256, T * CPR - 1);
                        const int row = blk * T + i / CPR, e0 = (i % CPR) * 8;
                        const int64_t token = (int64_t)b * p.S + (row - P);
                        const size_t off = (size_t)(token * a.H + h) * D + e0;
                        if constexpr (KIND == kInF16) {
                            raw[j][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(reinterpret_cast<const _Float16 *>(src) + off));
                        } else {
                            const u32x4 *at = reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint32_t *>(src) + off);
                            raw[j][0] = __builtin_nontemporal_load(at);
                            raw[j][1] = __builtin_nontemporal_load(at + 1);
                        }
                        if constexpr (KIND == kInI32) {
                            sc[j] = a.inp_scale[token];
                            ws[j][0] = *reinterpret_cast<const float4 *>(w + h * D + e0);
                            ws[j][1] = *reinterpret_cast<const float4 *>(w + h * D + e0 + 4);
                        }
                        if constexpr (!IS_V) {
                            const float4 *f = reinterpret_cast<const float4 *>(a.freq_cis + (size_t)(a.rope_row < 0 ? row : a.rope_row + (row - P)) * D + e0);
                            fr[j][0] = f[0];
                            fr[j][1] = f[1];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) {
                        if (n0 + j >= NI) continue;
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            if constexpr (KIND == kInF16) {
                                x[k] = (float)__builtin_bit_cast(half8, raw[j][0])[k];
                            } else if constexpr (KIND == kInF32) {
                                x[k] = __uint_as_float(raw[j][k / 4][k % 4]);
                            } else {
                                const float4 wk = ws[j][k / 4];
                                x[k] = __fmul_rn(__fmul_rn((float)(int)raw[j][k / 4][k % 4], sc[j]), k % 4 == 0 ? wk.x : (k % 4 == 1 ? wk.y : (k % 4 == 2 ? wk.z : wk.w)));
                            }
                        }
                        if constexpr (!IS_V) {
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                float r0, r1, r2, r3;
                                rope_pair(x[4 * k], x[4 * k + 1], fr[j][k].x, fr[j][k].y, r0, r1);
                                rope_pair(x[4 * k + 2], x[4 * k + 3], fr[j][k].z, fr[j][k].w, r2, r3);
                                x[4 * k] = r0; x[4 * k + 1] = r1; x[4 * k + 2] = r2; x[4 * k + 3] = r3;
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            kept[KEEP ? n0 + j : 0][k] = stored_half(x[k]); // (chunks behind the block repeat its last one)
                            absmax = fmaxf(absmax, fabsf((float)kept[KEEP ? n0 + j : 0][k]));
                        }
                    }
                }
            };
            auto by_kind = [&](auto v_tag) __attribute__((always_inline)) {
                if (p.in_kind == kInF16) load_block(std::integral_constant<int, kInF16>{}, v_tag);
                else if (p.in_kind == kInF32) load_block(std::integral_constant<int, kInF32>{}, v_tag);
                else load_block(std::integral_constant<int, kInI32>{}, v_tag);
            };
            if (is_v) by_kind(std::integral_constant<int, 1>{});
            else by_kind(std::integral_constant<int, 0>{});
        } else {
#pragma unroll KEEP ? NI : 1
            for (int n = 0; n < NI; ++n) {
                const int i = tid + n * 256;
                half8 x = half8{0, 0, 0, 0, 0, 0, 0, 0};
                if (EXACT || i < T * CPR) x = chunk(i);
#pragma unroll
                for (int j = 0; j < 8; ++j) absmax = fmaxf(absmax, fabsf((float)x[j]));
                if constexpr (KEEP) kept[n] = x;
            }
        }
        absmax = wave_max(absmax);
        if ((tid & 63) == 0) s_red[tid >> 6] = absmax;
        __syncthreads();
        absmax = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float f = quant_factor(absmax);
        uint2 *dst = reinterpret_cast<uint2 *>((is_v ? p.v8 : p.k8) + ((size_t)bh * a.L + (size_t)blk * T) * D);
#pragma unroll KEEP ? NI : 1
        for (int n = 0; n < NI; ++n) {
            const int i = tid + n * 256;
            if (!EXACT && i >= T * CPR) continue;
            const half8 x = KEEP ? kept[KEEP ? n : 0] : chunk(i);
            uint2 o;
            o.x = quantise4(x[0], x[1], x[2], x[3], f);
            o.y = quantise4(x[4], x[5], x[6], x[7], f);
            dst[i] = o;
        }
        if (tid == 0) (is_v ? p.v_scale : p.k_scale)[(size_t)bh * p.nblk + blk] = absmax / 127.0f;
    }
    if (nth == 0) {
        __syncthreads(); // the tail's old rows have been read
        const int r0 = max(last * T, P);
        for (int i = tid; i < (end - r0) * CPR; i += 256) {
            const int row = r0 + i / CPR, e0 = (i % CPR) * 8;
            *reinterpret_cast<half8 *>(tail + (size_t)(row - last * T) * D + e0) = new_chunk(row, e0);
        }
    }
}

// ---------------------------------------------------------------- read-back

// out_k, out_v [B,H,n,D] in O: integers * scale for complete blocks, the tail behind them, zeros behind a sequence's rows.
// grid = B*H * 2 * groups (the groups of 1024 chunks of one (b,h) fastest), block = 256; a lane writes 16 bytes.  Bound by the traffic, D bytes in and
// D * sizeof(O) out per row: 201 MB in 33 us, 6.2 TB/s.
struct Kv8ReadParams { // (a launch copies its arguments to the device: a third of Kv8Params is 0.2 us less)
    const int8_t *k8, *v8;
    const float *k_scale, *v_scale;
    const _Float16 *k_tail, *v_tail;
    const int32_t *rows_per_seq; // [B] or NULL
    int32_t H, L, T, t_shift;
};
template <typename O>
__global__ __launch_bounds__(256) void kv8_read_kernel(const Kv8ReadParams p, O *out_k, O *out_v, int n, int D, int groups)
{
    constexpr int VEC = 16 / (int)sizeof(O), NU = 4;
    typedef O vec __attribute__((ext_vector_type(VEC)));
    const int bh = blockIdx.x / groups >> 1, b = bh / p.H;
    const bool is_v = (blockIdx.x / groups & 1) != 0;
    // rows in the cache (a negative count: all zeros): where they end, not where the output does, the tail begins
    const int rows = min(p.rows_per_seq ? p.rows_per_seq[b] : n, p.L);
    const int rows8 = rows > 0 ? rows & ~(p.T - 1) : 0;
    const int8_t *src = (is_v ? p.v8 : p.k8) + (size_t)bh * p.L * D;
    const _Float16 *tail = (is_v ? p.v_tail : p.k_tail) + (size_t)bh * p.T * D;
    const float *scale = (is_v ? p.v_scale : p.k_scale) + (size_t)bh * (p.L >> p.t_shift);
    O *out = (is_v ? out_v : out_k) + (size_t)bh * n * D;
    const uint32_t CPR = D / VEC, total = (uint32_t)n * CPR; // (n * D stays below 2^31)
    const uint32_t i0 = (blockIdx.x % groups) * (256 * NU) + threadIdx.x;
    auto store = [&](const auto &x, const float (&sc)[NU]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const uint32_t i = i0 + u * 256;
            if (i >= total) return;
            const int row = (int)(i / CPR), e0 = (int)(i % CPR) * VEC;
            vec y;
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[j] = to_storage<O>(__fmul_rn((float)(int8_t)(x[u][j / 4] >> (8 * (j % 4))), sc[u]));
            if (row >= rows8) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] = (O)0;
                if (row < rows) {
                    const _Float16 *t = tail + (size_t)(row - rows8) * D + e0;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) y[j] = (O)t[j];
                }
            }
            *reinterpret_cast<vec *>(out + (size_t)i * VEC) = y; // (a non-temporal store: 36 us against 33)
        }
    };
    const uint32_t last = total - 1;
    if constexpr (VEC == 8) {
        typedef uint32_t words __attribute__((ext_vector_type(2)));
        words x[NU];
        float sc[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) { // rows that are no bytes repeat the first and are replaced below
            const uint32_t i = min(i0 + u * 256, last);
            const int row = (int)(i / CPR), e0 = (int)(i % CPR) * VEC, at = row < rows8 ? row : 0;
            x[u] = __builtin_nontemporal_load(reinterpret_cast<const words *>(src + (size_t)at * D + e0));
            sc[u] = scale[at >> p.t_shift];
        }
        __builtin_amdgcn_sched_barrier(0);
        store(x, sc);
    } else {
        uint32_t x[NU][1];
        float sc[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const uint32_t i = min(i0 + u * 256, last);
            const int row = (int)(i / CPR), e0 = (int)(i % CPR) * VEC, at = row < rows8 ? row : 0;
            x[u][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(src + (size_t)at * D + e0));
            sc[u] = scale[at >> p.t_shift];
        }
        __builtin_amdgcn_sched_barrier(0);
        store(x, sc);
    }
}

// ---------------------------------------------------------------- eviction

struct Kv8EvictParams {
    const int8_t *k8, *v8;
    const float *k_scale, *v_scale, *weights;
    const _Float16 *k_tail, *v_tail;
    int8_t *k8_to, *v8_to;
    float *k_scale_to, *v_scale_to, *weights_to;
    _Float16 *k_tail_to, *v_tail_to; // NULL: the tails stay where they are
    int32_t *kept;                // [B*H, keep] source blocks in ascending order, -1 behind the last
    int32_t *rows_to;             // [B]
    const int32_t *rows_per_seq;  // [B] or NULL
    int32_t rows, B, H, D, T, t_shift, nblk, nblk_to, keep, recent;
};

// Rows of sequence b before the eviction; -1 where the count lies outside the cache (nothing is moved then).
__device__ __forceinline__ int evict_rows(const Kv8EvictParams &p, int b)
{
    const int r = p.rows_per_seq ? p.rows_per_seq[b] : p.rows;
    return r < 0 || r > p.nblk * p.T ? -1 : r;
}

// Order-preserving unsigned image of a weight: larger weight, larger key; NaN below everything, -0 = +0.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of a flag over the NT threads; total: the number of flags set.
template <int NT>
__device__ __forceinline__ int block_rank(bool flag, int *s_cnt, int &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned long long bal = __ballot(flag);
    __syncthreads(); // s_cnt is free
    if (lane == 0) s_cnt[wave] = __popcll(bal);
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) before += s_cnt[w];
        total += s_cnt[w];
    }
    return before + __popcll(bal & ((1ull << lane) - 1ull));
}

// Which blocks of (b,h) stay: the last `recent` and, of the rest, those of the largest weight, ties to the lowest block.  Few
// candidates count for each how many come before it.  Of many, the weight of the last one that stays is found by four passes over
// the bits of the keys, eight at a time (a histogram in LDS each).  The list is then written in ascending order, and scales and
// weights move with it; in place, an entry moves to its own or a lower slot: NT entries are read before they are written.
constexpr int kCountedBlocks = 64; // (each comes down to 16 reads of four keys)
struct SelectShared {
    alignas(16) uint32_t key[kCountedBlocks]; // read four at a time
    int hist[256];
    int cnt[16];
    uint32_t pick[2]; // threshold byte, entries still wanted at it
};
static_assert(alignof(SelectShared) >= sizeof(uint4) && kCountedBlocks % 4 == 0, "the keys are read as uint4");
template <int NT>
__device__ __forceinline__ void select_blocks(const Kv8EvictParams &p, int bh, int rows, int *s_list, SelectShared &sh)
{
    const int b = bh / p.H, tid = threadIdx.x;
    const int n = rows < 0 ? 0 : rows >> p.t_shift;
    const int keep = min(p.keep, n), recent = min(p.recent, keep);
    const int cand = n - recent, want = keep - recent; // the first `cand` blocks compete for `want` places
    const float *w = p.weights + (size_t)bh * p.nblk, *ks = p.k_scale + (size_t)bh * p.nblk, *vs = p.v_scale + (size_t)bh * p.nblk;
    const bool all = want >= cand, none = want <= 0, counted = cand <= kCountedBlocks;
    // the first NT blocks' values, and the open block's
    float ws = 0.f, ksc = 0.f, vsc = 0.f, w_open = 0.f;
    if (tid < n) {
        ws = w[tid];
        ksc = ks[tid];
        vsc = vs[tid];
    }
    const int open = rows < 0 ? 0 : rows & (p.T - 1);
    if (tid == 0 && open) w_open = w[n];
    uint32_t prefix = 0, mask = 0;
    int left = want;
    bool chosen = false;
    if (!all && !none && counted) {
        if (tid < kCountedBlocks) sh.key[tid] = tid < cand ? weight_key(ws) : 0u;
        __syncthreads();
        if (tid < cand) {
            const uint32_t k = sh.key[tid];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < cand; i += 4) { // (keys behind the last are no larger than any, and come later)
                const uint4 y = *reinterpret_cast<const uint4 *>(&sh.key[i]);
                rank += (int)(y.x > k || (y.x == k && i < tid)) + (int)(y.y > k || (y.y == k && i + 1 < tid)) +
                        (int)(y.z > k || (y.z == k && i + 2 < tid)) + (int)(y.w > k || (y.w == k && i + 3 < tid));
            }
            chosen = rank < want;
        }
    } else if (!all && !none) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < cand; i += NT) {
                const uint32_t k = weight_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&sh.hist[(k >> shift) & 255u], 1);
            }
            __syncthreads();
            if (tid < 64) { // the largest byte whose keys and all larger ones are enough: one wave, four bytes a lane
                const int d3 = sh.hist[255 - 4 * tid], d2 = sh.hist[254 - 4 * tid], d1 = sh.hist[253 - 4 * tid], d0 = sh.hist[252 - 4 * tid];
                int sum = d3 + d2 + d1 + d0, incl = sum;
#pragma unroll
                for (int o = 1; o < 64; o *= 2) {
                    const int y = __shfl_up(incl, o);
                    if (tid >= o) incl += y;
                }
                const int above = incl - sum;
                if (above < left && incl >= left) {
                    int byte = 255 - 4 * tid, at = above;
                    if (at + d3 < left) { at += d3; --byte; if (at + d2 < left) { at += d2; --byte; if (at + d1 < left) { at += d1; --byte; } } }
                    sh.pick[0] = (uint32_t)byte;
                    sh.pick[1] = (uint32_t)(left - at);
                }
            }
            __syncthreads();
            prefix |= sh.pick[0] << shift;
            mask |= 255u << shift;
            left = (int)sh.pick[1];
            __syncthreads();
        }
    }
    int *list = p.kept + (size_t)bh * p.keep;
    int placed = 0, equal = 0;
    for (int base = 0; base < n; base += NT) {
        const int i = base + tid;
        if (base > 0 && i < n) {
            ws = w[i];
            ksc = ks[i];
            vsc = vs[i];
        }
        bool stay = i < n && (i >= cand || all);
        if (!all && !none && counted) {
            stay = stay || (base == 0 && chosen); // (NT >= kCountedBlocks: every candidate is in the first trip)
        } else if (!all && !none) { // keys above `prefix` stay, and the first `left` equal to it
            const uint32_t k = i < cand ? weight_key(ws) : 0u;
            const bool tie = i < cand && k == prefix;
            int n_tie;
            const int tie_rank = equal + block_rank<NT>(tie, sh.cnt, n_tie);
            equal += n_tie;
            stay = stay || (i < cand && (k > prefix || (tie && tie_rank < left)));
        }
        int n_stay;
        const int at = placed + block_rank<NT>(stay, sh.cnt, n_stay); // its barriers: read before any slot of this trip is written
        if (stay) {
            list[at] = i;
            if (s_list) s_list[at] = i;
            p.weights_to[(size_t)bh * p.nblk_to + at] = ws;
            p.k_scale_to[(size_t)bh * p.nblk_to + at] = ksc;
            p.v_scale_to[(size_t)bh * p.nblk_to + at] = vsc;
        }
        placed += n_stay;
    }
    for (int i = keep + tid; i < p.keep; i += NT) list[i] = -1;
    if (tid == 0) {
        if (open && keep < p.nblk_to) p.weights_to[(size_t)bh * p.nblk_to + keep] = w_open;
        if (bh % p.H == 0) p.rows_to[b] = rows < 0 ? -1 : (keep << p.t_shift) + open;
    }
}

// Moves one 16-byte column of the listed blocks of K or V.  In place nothing but its own column can stand in its way, and it
// moves the blocks in ascending order, NB of them read before the first is written (a block moves to its own or a lower slot).
template <int NB>
__device__ __forceinline__ void move_column(const Kv8EvictParams &p, int bh, bool is_v, int col, int keep, const int *list)
{
    const int cols = p.T * p.D / 16;
    const u32x4 *src = reinterpret_cast<const u32x4 *>((is_v ? p.v8 : p.k8) + (size_t)bh * p.nblk * p.T * p.D) + col;
    u32x4 *dst = reinterpret_cast<u32x4 *>((is_v ? p.v8_to : p.k8_to) + (size_t)bh * p.nblk_to * p.T * p.D) + col;
    for (int r0 = 0; r0 < keep; r0 += NB) {
        u32x4 x[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) x[u] = __builtin_nontemporal_load(src + (size_t)list[min(r0 + u, keep - 1)] * cols);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < NB; ++u)
            if (r0 + u < keep) __builtin_nontemporal_store(x[u], dst + (size_t)(r0 + u) * cols);
    }
}
// The open rows of K or V into a cache with tails of its own, by NT threads.
template <int NT>
__device__ __forceinline__ void move_tail(const Kv8EvictParams &p, int bh, bool is_v, int rows)
{
    _Float16 *tail_to = is_v ? p.v_tail_to : p.k_tail_to;
    if (!tail_to) return;
    const half8 *src = reinterpret_cast<const half8 *>((is_v ? p.v_tail : p.k_tail) + (size_t)bh * p.T * p.D);
    half8 *dst = reinterpret_cast<half8 *>(tail_to + (size_t)bh * p.T * p.D);
    for (int i = threadIdx.x; i < (rows & (p.T - 1)) * (p.D / 8); i += NT) dst[i] = src[i];
}

// The selection as a launch of its own: grid = B*H, block = 256.
__global__ __launch_bounds__(256) static void kv8_select_kernel(const Kv8EvictParams p)
{
    __shared__ SelectShared sh;
    select_blocks<256>(p, blockIdx.x, evict_rows(p, blockIdx.x / p.H), nullptr, sh);
}

// Moves the listed blocks: grid = B*H * 2 * slices of a block (fastest), block = 256, a thread per column.  32 (b,h) of 512 KB: 14 us
// with the selection.
__global__ __launch_bounds__(256) static void kv8_move_kernel(const Kv8EvictParams p, int slices)
{
    const int bh = blockIdx.x / slices >> 1, slice = blockIdx.x % slices;
    const bool is_v = (blockIdx.x / slices & 1) != 0;
    const int rows = evict_rows(p, bh / p.H);
    if (rows < 0) return;
    const int col = slice * 256 + threadIdx.x;
    if (col < p.T * p.D / 16) move_column<8>(p, bh, is_v, col, min(p.keep, rows >> p.t_shift), p.kept + (size_t)bh * p.keep);
    if (slice == 0) move_tail<256>(p, bh, is_v, rows);
}

// Both in one launch, where a workgroup has little to move or there is one for every compute unit: grid = B*H, block = kEvictThreads.
// Bound by the traffic: 1.07 GB read and written in 190 us, 5.6 TB/s (a plain copy of half of that: 5.35; in two launches 200,
// there with stores that go through the caches 212, with 4 or 16 blocks at a time 210 / 202).
constexpr int kEvictThreads = 1024, kEvictListCap = 1024;
__global__ __launch_bounds__(kEvictThreads) static void kv8_evict_kernel(const Kv8EvictParams p)
{
    __shared__ SelectShared sh;
    __shared__ int s_list[kEvictListCap];
    const int bh = blockIdx.x, rows = evict_rows(p, bh / p.H);
    select_blocks<kEvictThreads>(p, bh, rows, s_list, sh);
    if (rows < 0) return; // (uniform)
    __syncthreads(); // the list
    const int keep = min(p.keep, rows >> p.t_shift), cols = p.T * p.D / 16;
    for (int c = threadIdx.x; c < 2 * cols; c += kEvictThreads) {
        const bool is_v = c >= cols;
        if (p.keep > 4) move_column<8>(p, bh, is_v, is_v ? c - cols : c, keep, s_list);
        else move_column<4>(p, bh, is_v, is_v ? c - cols : c, keep, s_list);
    }
    move_tail<kEvictThreads>(p, bh, false, rows);
    move_tail<kEvictThreads>(p, bh, true, rows);
}

} // namespace flattn
