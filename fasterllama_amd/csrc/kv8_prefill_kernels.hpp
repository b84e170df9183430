// Prompt phase over the 8-bit cache on the matrix cores (size_per_head 32, 64, 96, 128).
//
// Same shape as the fp16 caches' kernel: a workgroup owns 128 queries of one (b,h), 32 per wave, and walks the keys 32 at a
// time through LDS; S^T = K Q^T leaves 16 probabilities of one query in every lane, in the operand layout of O^T = V^T P^T.
// What the 8 bits change:
//   operands   a byte is an exact fp16 number, so K and V enter v_mfma_f32_32x32x16_f16 as they are stored and the block's
//              scale (uniform over a 32-key tile) stays outside: K's multiplies the score where the softmax scale does, V's
//              goes into the exponent of the weight, e^(s - m) * vs / 2^r = 2^(s' - m' + log2(vs) - r), and costs nothing
//              per score either.  A query's references m and r follow the largest PRODUCT of weight and scale met so far: a
//              block of large values that gets no weight, or one of zeros, must not decide how finely the others' are held;
//   precision  queries and weights are fp16 PAIRS, value + remainder (22 bits), twice the matrix instructions of single
//              values, so that the output keeps the accuracy of 32-bit arithmetic (2e-7 of the result at the 7B shapes;
//              weights rounded once to fp16 would leave 1.4e-4).  A query is scaled by a power of two so that its largest
//              element lies in [256, 512), a weight by 2^7: remainders stay clear of fp16's smallest steps;
//   loads      a tile is half the bytes: one 16-byte chunk of K and of V per thread (D = 128), widened to fp16 on the way
//              into LDS by all four waves together.
// Bound by the matrix instructions and what stands between them: B=1, S=4096, 32 heads, causal: 288 us, 292 GFLOP executed (the
// pairs counted twice) = 1.0 PFLOP/s, matrix pipe busy 53 % of the cycles; B=8, S=1024: 193 us, 0.75 PFLOP/s, of which 63 us
// are what a workgroup does before and after its tiles.  Taken out one at a time (S=4096 / S=1024): the remainders' products
// 219 / 163 us, the widening 272 / 196, the exponentials 268 / 194, reading and rotating the queries 265 / 168.
#pragma once

#include "kv8_kernels.hpp"

#pragma clang fp contract(off)

namespace flattn {

// Weights times V scale enter the second product relative to a query's largest such product, times 2^7; kLazyMax = 8 more stay below
// 65504.  The remainder's smallest step is 2^-24: a weight is held to 2^-22 of itself or to 2^-32 of that largest product.
constexpr float kKv8WeightExp = 7.0f;
// A block's scale is 0 or lies in [2^-31, 2^10) (fp16's steps over 127).  Zeros count as 2^-80: small enough to leave the reference to the
// others where they take e^-50 of the weight, while the sum of the weights, in units of the reference's score, stays below 2^127.
constexpr int kKv8LeastScaleExp = -80;

struct Kv8PromptParams {
    Kv8Params k;
    PrefillParams f;      // mask, tile classes, B, H, L, S, start_pos
    half8 *q_pairs;       // workspace: rotated query operands of the last queries, for the block weights; or NULL
    float *q_factor;      // [B*H, query blocks of 32, 32] with them
    int32_t kept_blocks;  // 32-query blocks of a sequence that they have room for; which ones: first_kept_block
    int32_t key_splits;   // workgroups that share the keys of a (query block, head); > 1: partials, merged by kv8_prompt_merge_kernel
    int32_t part_rows;    // queries per partial: 128, or the prompt's where it is shorter
    float *part_o;        // workspace [B*H * query blocks * splits, part_rows, D]: sums of weight * value, not normalised
    float2 *part_ml;      // [.., part_rows]: (reference maximum, sum of weights)
};

// Four signed bytes as fp16: 1024 + (b ^ 128) is the fp16 with that low byte, minus 1152 leaves b, exactly.
__device__ __forceinline__ void widen4(uint32_t x, half2v &lo, half2v &hi)
{
    const uint32_t u = x ^ 0x80808080u;
    const half2v off = {(_Float16)-1152.f, (_Float16)-1152.f};
    lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
}

// Classes of a key tile for the four 32-query sub-blocks of a 128-query block.  A short context is not classified (a launch of
// its own costs more than reading its mask): every tile is kTileMixed, that of a sub-block behind the prompt kTileSkip.
constexpr int kUnclassifiedKeys = 128;
__device__ __forceinline__ uint32_t prompt_class_word(const PrefillParams &f, int qb, int t, int NT)
{
    if (f.tile_class || f.class_table) return tile_class_word(f, qb, t, NT);
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (qb * kPrefillQueriesPerBlock + 32 * k < f.S) w |= kTileMixed << (8 * k);
    return w;
}

// The first 32-query block with one of the last weight_queries of a sequence's `tokens` queries.
__device__ __forceinline__ int first_kept_block(const Kv8Params &p, int tokens) { return max(tokens - p.weight_queries, 0) / 32; }

__device__ __forceinline__ void wave_lds_sync() // orders this wave's LDS writes and reads
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int D, bool HAS_MASK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 8)))
void kv8_prefill_attn_kernel(const Kv8PromptParams pp)
{
    constexpr int BN = kPrefillKeysPerStep; // 32
    constexpr int LDK = D + 8;                       // halfs; rows start 4 banks apart (128-bit operand reads)
    constexpr int LDV = D == 96 ? D + 48 : D + 32;   // halfs; for the transposing reads, as the fp16 caches' kernel
    constexpr int NC = D / 16, NDT = D / 32;
    constexpr int NCH = BN * D / 16;                 // 16-byte chunks of a byte tile
    constexpr int LPT = (2 * NCH + 255) / 256;       // chunks per thread: K's first, then V's
    constexpr int CPR8 = D / 16;                     // chunks per row
    constexpr int LDQ = D + 8, HALF_D = D >= 128 ? 64 : 32, LDO = HALF_D + 4;
    constexpr int TILE_HALFS = 2 * BN * (LDK + LDV), Q_HALFS = kPrefillQueriesPerBlock * LDQ, O_HALFS = kPrefillQueriesPerBlock * LDO * 2;
    constexpr int SMEM_HALFS = TILE_HALFS > Q_HALFS ? (TILE_HALFS > O_HALFS ? TILE_HALFS : O_HALFS) : (Q_HALFS > O_HALFS ? Q_HALFS : O_HALFS);
    __shared__ __attribute__((aligned(16))) _Float16 smem[SMEM_HALFS];
    __shared__ uint32_t s_list[HAS_MASK ? kTileListCap : 1];
    __shared__ int s_wave_cnt[4];
    __shared__ uint32_t s_qmax[kPrefillQueriesPerBlock];
    _Float16 (*sK)[BN][LDK] = reinterpret_cast<_Float16 (*)[BN][LDK]>(smem);
    _Float16 (*sV)[BN][LDV] = reinterpret_cast<_Float16 (*)[BN][LDV]>(smem + 2 * BN * LDK);

    const Kv8Params &p = pp.k;
    const Params &a = p.a;
    const PrefillParams &pf = pp.f;
    const int BH = a.B * a.H, S = p.S, P = a.start_pos, L = a.L;
    int qb, bh;
    const int QB = (S + kPrefillQueriesPerBlock - 1) / kPrefillQueriesPerBlock, KS = pp.key_splits, split = (int)blockIdx.x / (QB * BH);
    prefill_block_to_tile((int)blockIdx.x % (QB * BH), BH, QB, HAS_MASK, qb, bh);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tokens = kv8_prompt_tokens(p, bh / a.H);
    if (qb * kPrefillQueriesPerBlock >= tokens) { // none of the sequence's own (uniform)
        if (KS > 1) return; // (the merge sees to them)
        const int n = min(kPrefillQueriesPerBlock, S - qb * kPrefillQueriesPerBlock);
        const float x = kv8_no_query(tokens);
        float4 *dst = reinterpret_cast<float4 *>(a.out + ((size_t)bh * S + qb * kPrefillQueriesPerBlock) * D);
        for (int i = tid; i < n * (D / 4); i += 256) dst[i] = make_float4(x, x, x, x);
        return;
    }
    const int ctx = P + tokens, ctx8 = ctx & ~(p.T - 1); // rows [0, ctx8) are bytes, [ctx8, ctx) wait in the tail
    const int NT = (ctx + BN - 1) / BN, class_ld = (P + S + BN - 1) / BN;
    const int qi = lane & 31, hf = lane >> 5;
    const int q_row = qb * kPrefillQueriesPerBlock + wave * 32 + qi;

    auto build_list = [&](int c0, int c1, bool have_first, uint32_t w_first) __attribute__((always_inline)) -> int {
        return build_tile_list(pf, qb, c0, c1, class_ld, have_first, w_first, s_list, s_wave_cnt);
    };
    // entry i of this workgroup's share, which starts at `share` of the pass's list
    int share = 0;
    auto list_entry = [&](int c0, int i) __attribute__((always_inline)) -> uint32_t {
        if constexpr (HAS_MASK) return s_list[share + i];
        else return (uint32_t)(c0 + share + i) << 8 | 0x55u;
    };
    auto take_share = [&](int n) __attribute__((always_inline)) -> int { // of n listed tiles
        if (KS == 1) return n;
        share = (int)((int64_t)n * split / KS);
        return (int)((int64_t)n * (split + 1) / KS) - share;
    };

    // global -> registers (fetch), registers -> LDS (commit) of a key tile.  A tile of the tail — fp16 rows, twice the loads, the
    // last few tiles of the context — is loaded where it is committed: registers for both kinds would have to be merged
    // behind the request, and the merge waits for the loads.  Its rows behind the context become zeros.
    const size_t row_off = (size_t)bh * L * D, tail_off = (size_t)bh * p.T * D;
    const float *ks_at = p.k_scale + (size_t)bh * p.nblk, *vs_at = p.v_scale + (size_t)bh * p.nblk;
    u32x4 stage[LPT];
    float stage_ks = 1.f, stage_vs = 1.f; // the tile's scales travel with it
    auto fetch = [&](int t) __attribute__((always_inline)) {
        if (t * BN >= ctx8) return; // uniform
        stage_ks = ks_at[t * BN >> p.t_shift];
        stage_vs = vs_at[t * BN >> p.t_shift];
#pragma unroll
        for (int j = 0; j < LPT; ++j) {
            const bool is_v = (wave + 4 * j) * 64 >= NCH; // uniform: NCH is a multiple of 64
            const int i = tid + j * 256 - (is_v ? NCH : 0);
            if (2 * NCH % 256 == 0 || (wave + 4 * j) * 64 < 2 * NCH)
                stage[j] = *reinterpret_cast<const u32x4 *>((is_v ? p.v8 : p.k8) + row_off + (size_t)t * (BN * D) + i * 16);
        }
    };
    float next_ks = 1.f, next_vs = 1.f;
    auto commit = [&](int t, int buf) __attribute__((always_inline)) {
        const bool tail = t * BN >= ctx8;
        next_ks = tail ? 1.f : __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(stage_ks))); // tail rows are values
        next_vs = tail ? 1.f : __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(stage_vs)));
#pragma unroll
        for (int j = 0; j < LPT; ++j) {
            const bool is_v = (wave + 4 * j) * 64 >= NCH;
            const int i = tid + j * 256 - (is_v ? NCH : 0);
            const int r = i / CPR8, e0 = (i % CPR8) * 16;
            if (2 * NCH % 256 == 0 || (wave + 4 * j) * 64 < 2 * NCH) {
                half8 *dst = reinterpret_cast<half8 *>(is_v ? &sV[buf][r][e0] : &sK[buf][r][e0]);
                if (!tail) {
                    half2v h[8];
                    widen4(stage[j][0], h[0], h[1]);
                    widen4(stage[j][1], h[2], h[3]);
                    widen4(stage[j][2], h[4], h[5]);
                    widen4(stage[j][3], h[6], h[7]);
                    half8 y0, y1;
#pragma unroll
                    for (int c = 0; c < 8; ++c) { y0[c] = h[c / 2][c % 2]; y1[c] = h[4 + c / 2][c % 2]; }
                    dst[0] = y0;
                    dst[1] = y1;
                } else {
                    const int row = t * BN + r - ctx8;
                    half8 y0 = half8{0, 0, 0, 0, 0, 0, 0, 0}, y1 = y0;
                    if (row < ctx - ctx8) {
                        const half8 *src = reinterpret_cast<const half8 *>((is_v ? p.v_tail : p.k_tail) + tail_off + (size_t)row * D + e0);
                        y0 = src[0];
                        y1 = src[1];
                    }
                    dst[0] = y0;
                    dst[1] = y1;
                }
            }
        }
    };

    const int first_c1 = min(kTileListCap, NT);
    if (split == 0) fetch(0); // a guess at the first listed tile: right without a mask and under every causal one
    uint32_t w_first = 0;
    if constexpr (HAS_MASK) {
        if (tid < first_c1) w_first = prompt_class_word(pf, qb, tid, class_ld);
    }

    // The rotated queries as fp16 pairs in operand layout, by way of LDS: every wave its own 32 (see the fp16 caches'
    // kernel for the data path), scaled by a power of two that comes back in qc.
    half8 qhi[NC], qlo[NC];
    float qc; // softmax scale * log2 e / that power, of this lane's query
    {
        constexpr int CPR = D / 8, QPL = 32 * CPR / 64;
        constexpr bool FIXED_COL = 64 % CPR == 0;
        constexpr int RPI = FIXED_COL ? 64 / CPR : 1;
        auto q_rl = [&](int j) __attribute__((always_inline)) -> int { return FIXED_COL ? lane / CPR + j * RPI : (lane + 64 * j) / CPR; };
        auto q_cc = [&](int j) __attribute__((always_inline)) -> int { return FIXED_COL ? lane % CPR : (lane + 64 * j) % CPR; };
        const int b = bh / a.H, h = bh % a.H, row0 = a.rope_row < 0 ? P : a.rope_row;
        const int q_first = qb * kPrefillQueriesPerBlock + wave * 32;
        _Float16 *const sq = smem + wave * 32 * LDQ;
        float x[QPL][8];
        auto load_queries = [&](auto kind_tag) __attribute__((always_inline)) {
            constexpr int KIND = decltype(kind_tag)::value;
            constexpr int BATCH = KIND != kInF16 && QPL > 1 ? QPL / 2 : QPL;
#pragma unroll
            for (int j0 = 0; j0 < QPL; j0 += BATCH) {
                u32x4 raw[BATCH][KIND == kInF16 ? 1 : 2];
                float4 f[BATCH][2], w[KIND == kInI32 ? BATCH : 1][2];
                float sc[KIND == kInI32 ? BATCH : 1];
#pragma unroll
                for (int jj = 0; jj < BATCH; ++jj) { // rows past the prompt read its last one and are zeroed below
                    const int cc = q_cc(j0 + jj), q = min(q_first + q_rl(j0 + jj), S - 1);
                    const int64_t token = (int64_t)b * S + q;
                    const size_t off = (size_t)(token * a.H + h) * D + cc * 8;
                    if constexpr (KIND == kInF16) {
                        raw[jj][0] = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const _Float16 *>(a.q) + off);
                    } else {
                        const u32x4 *src = reinterpret_cast<const u32x4 *>(reinterpret_cast<const float *>(a.q) + off);
                        raw[jj][0] = src[0];
                        raw[jj][1] = src[1];
                    }
                    if constexpr (KIND == kInI32) {
                        sc[jj] = a.inp_scale[token];
                        w[jj][0] = *reinterpret_cast<const float4 *>(a.wq_scale + h * D + cc * 8);
                        w[jj][1] = *reinterpret_cast<const float4 *>(a.wq_scale + h * D + cc * 8 + 4);
                    }
                    const float4 *fr = reinterpret_cast<const float4 *>(a.freq_cis + (size_t)(row0 + q) * D + cc * 8);
                    f[jj][0] = fr[0];
                    f[jj][1] = fr[1];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int jj = 0; jj < BATCH; ++jj) {
                    float v[8];
                    if constexpr (KIND == kInF16) {
                        const half8 y = __builtin_bit_cast(half8, raw[jj][0]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = (float)y[i];
                    } else if constexpr (KIND == kInF32) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(raw[jj][i / 4][i % 4]);
                    } else {
                        const float ws[8] = {w[jj][0].x, w[jj][0].y, w[jj][0].z, w[jj][0].w, w[jj][1].x, w[jj][1].y, w[jj][1].z, w[jj][1].w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fmul_rn((float)(int)raw[jj][i / 4][i % 4], sc[jj]), ws[i]);
                    }
                    const bool valid = q_first + q_rl(j0 + jj) < tokens;
                    float *o = x[j0 + jj];
                    rope_pair(v[0], v[1], f[jj][0].x, f[jj][0].y, o[0], o[1]);
                    rope_pair(v[2], v[3], f[jj][0].z, f[jj][0].w, o[2], o[3]);
                    rope_pair(v[4], v[5], f[jj][1].x, f[jj][1].y, o[4], o[5]);
                    rope_pair(v[6], v[7], f[jj][1].z, f[jj][1].w, o[6], o[7]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = valid ? o[i] : 0.f;
                }
            }
        };
        if (p.in_kind == kInF16) load_queries(std::integral_constant<int, kInF16>{});
        else if (p.in_kind == kInF32) load_queries(std::integral_constant<int, kInF32>{});
        else load_queries(std::integral_constant<int, kInI32>{});

        // largest |element| of every query (bit patterns of non-negative floats order as integers)
        uint32_t *const qmax = s_qmax + wave * 32;
        if (lane < 32) qmax[lane] = 0u;
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < QPL; ++j) {
            float top = 1e-30f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
            if constexpr (FIXED_COL) {
                top = fmaxf(top, dpp_move<0xB1>(top));
                top = fmaxf(top, dpp_move<0x4E>(top));
                if constexpr (CPR >= 8) top = fmaxf(top, dpp_move<0x141>(top));
                if constexpr (CPR >= 16) top = fmaxf(top, dpp_move<0x140>(top));
                if (lane % CPR == 0) qmax[q_rl(j)] = __float_as_uint(top);
            } else {
                atomicMax(&qmax[q_rl(j)], __float_as_uint(top));
            }
        }
        wave_lds_sync();
        auto power = [&](uint32_t top_bits) __attribute__((always_inline)) -> float { // 2^(8 - floor(log2 top))
            return __uint_as_float((uint32_t)(127 + 8 + 127 - (int)(top_bits >> 23)) << 23);
        };
        half8 lo_keep[QPL];
#pragma unroll
        for (int j = 0; j < QPL; ++j) {
            const float f = power(qmax[q_rl(j)]);
            half8 hq;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[j][i] * f;
                hq[i] = (_Float16)y;
                lo_keep[j][i] = (_Float16)(y - (float)hq[i]);
            }
            *reinterpret_cast<half8 *>(sq + q_rl(j) * LDQ + q_cc(j) * 8) = hq;
        }
        wave_lds_sync();
#pragma unroll
        for (int c = 0; c < NC; ++c) qhi[c] = *reinterpret_cast<const half8 *>(sq + qi * LDQ + 16 * c + 8 * hf);
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < QPL; ++j) *reinterpret_cast<half8 *>(sq + q_rl(j) * LDQ + q_cc(j) * 8) = lo_keep[j];
        wave_lds_sync();
#pragma unroll
        for (int c = 0; c < NC; ++c) qlo[c] = *reinterpret_cast<const half8 *>(sq + qi * LDQ + 16 * c + 8 * hf);
        const uint32_t e = qmax[qi] >> 23; // biased exponent of the largest element
        qc = a.scale * kLog2e * __uint_as_float((uint32_t)((int)e - 8) << 23);
        const int block = q_first / 32 - first_kept_block(p, tokens);
        if (pp.q_pairs && split == 0 && block >= 0 && q_first < tokens) { // kept for the block weights
            half8 *dst = pp.q_pairs + ((size_t)bh * pp.kept_blocks + block) * (2 * NC * 64) + lane;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                dst[c * 64] = qhi[c];
                dst[(NC + c) * 64] = qlo[c];
            }
            if (hf == 0) pp.q_factor[((size_t)bh * pp.kept_blocks + block) * 32 + qi] = qc;
        }
    }
    if constexpr (!HAS_MASK) __syncthreads(); // the slices lie in the tile buffers (with a mask the list's barriers see to it)
    int n_first = first_c1;
    if constexpr (HAS_MASK) n_first = build_list(0, first_c1, true, w_first);
    n_first = take_share(n_first);
    if (n_first > 0) {
        const int t_first = (int)(__builtin_amdgcn_readfirstlane(list_entry(0, 0)) >> 8);
        if (t_first != 0 || split != 0) fetch(t_first);
    }

    floatx16 ot[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) ot[dt][v] = 0.f;
    // Per query: weights are 2^(s' - m), l is their sum, output accumulators are in units of 2^r (a whole number).
    float m = kMaxFloor * kLog2e, r = (float)kKv8LeastScaleExp, l = 0.f;
    const int vrow = 4 * hf + ((lane & 15) >> 2), vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int c = 0; c < NC; ++c) asm volatile("" : "+v"(qhi[c]), "+v"(qlo[c]));

    for (int c0 = 0; c0 < NT; c0 += kTileListCap) {
        const int c1 = min(c0 + kTileListCap, NT);
        int n = c1 - c0;
        if (c0 == 0) {
            n = n_first;
        } else {
            if constexpr (HAS_MASK) n = build_list(c0, c1, false, 0u); // ends with a barrier
            else __syncthreads();
            n = take_share(n);
        }
        if (n == 0) continue;
        uint32_t e0 = __builtin_amdgcn_readfirstlane(list_entry(c0, 0));
        uint32_t e1 = n > 1 ? __builtin_amdgcn_readfirstlane(list_entry(c0, 1)) : 0u;
        uint32_t e2 = n > 2 ? __builtin_amdgcn_readfirstlane(list_entry(c0, 2)) : 0u;
        if (c0 > 0) fetch((int)(e0 >> 8));
        commit((int)(e0 >> 8), 0);
        if (n > 1) fetch((int)(e1 >> 8));
        auto tile_step = [&](int i, auto buf_tag) __attribute__((always_inline)) {
            constexpr int buf = decltype(buf_tag)::value;
            const int t = (int)(e0 >> 8), k0 = t * BN;
            const float ks = next_ks, vs_tile = next_vs; // committed with tile t
            __syncthreads(); // tile t is visible; every wave is done with the other buffer
            uint32_t tc = kTileZero;
            if constexpr (HAS_MASK) tc = __builtin_amdgcn_readfirstlane((e0 >> (2 * wave)) & 3u);
            const bool special = tc != kTileSkip && (k0 + BN > ctx || tc >= kTileMixed);
            float mk[16];
            if constexpr (HAS_MASK) {
                if (special && tc == kTileMixed) { // before the next tile is requested: loads return in order
                    const float *mrow = pf.attn_mask + (size_t)(P + min(q_row, S - 1)) * pf.mask_ld;
#pragma unroll
                    for (int v = 0; v < 16; ++v) mk[v] = mrow[min(k0 + 8 * (v / 4) + 4 * hf + (v % 4), ctx - 1)];
                }
            }
            if (i + 1 < n) {
                commit((int)(e1 >> 8), buf ^ 1);
                if (i + 2 < n) fetch((int)(e2 >> 8));
            }
            if (tc != kTileSkip) {
                floatx16 st;
#pragma unroll
                for (int v = 0; v < 16; ++v) st[v] = 0.f;
                // Operands are read from LDS one step ahead of the products that use them, the scheduler held to it: left alone
                // it reads them right before, and every few products wait out an LDS round trip.
                half8 kc[2][2];
                auto k_stage = [&](int which, int c) __attribute__((always_inline)) {
                    kc[which][0] = *reinterpret_cast<const half8 *>(&sK[buf][qi][16 * c + 8 * hf]);
                    kc[which][1] = *reinterpret_cast<const half8 *>(&sK[buf][qi][16 * (c + 1) + 8 * hf]);
                };
                k_stage(0, 0);
#pragma unroll
                for (int c = 0; c < NC; c += 2) {
                    if (c + 2 < NC) k_stage((c / 2 + 1) & 1, c + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kc[(c / 2) & 1][cc], qlo[c + cc], st, 0, 0, 0);
                        st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kc[(c / 2) & 1][cc], qhi[c + cc], st, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                half4 vst[2][4];
                auto v_stage = [&](int which, int dt) __attribute__((always_inline)) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        vst[which][2 * u] = lds_read_tr16(&sV[buf][16 * u + vrow][32 * dt + vcol]);
                        vst[which][2 * u + 1] = lds_read_tr16(&sV[buf][16 * u + 8 + vrow][32 * dt + vcol]);
                    }
                };
                v_stage(0, 0);
                __builtin_amdgcn_sched_barrier(0);
                float cs = qc * ks; // raw product -> base-2 score
                if (special) {
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const int key = 8 * (v / 4) + 4 * hf + (v % 4);
                        float s = st[v] * cs;
                        if constexpr (HAS_MASK) {
                            if (tc == kTileMixed) s = fmaf(mk[v], kLog2e, s);
                            if (tc == kTileDiag && key > qi) s = -__builtin_inff();
                        }
                        st[v] = k0 + key >= ctx ? -__builtin_inff() : s;
                    }
                    cs = 1.f;
                }
                // log2 of the block's scale as a whole number and a fraction, so that its differences to r stay exact
                const uint32_t vbits = __builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(vs_tile, __builtin_ldexpf(1.0f, kKv8LeastScaleExp))));
                const float vexp = (float)((int)(vbits >> 23) - 127), vfrac = __builtin_amdgcn_logf(__uint_as_float((vbits & 0x7fffffu) | 0x3f800000u));
                const float mx = cross_half_max(max16(st)) * cs;
                const float over = (mx - m) + (vexp - r) + vfrac; // of this tile's largest product over the reference (-inf: all masked)
                if (__ballot(over > kLazyMax) != 0ull) { // wave-uniform
                    const float m_new = over > 0.f ? mx : m, r_new = over > 0.f ? vexp : r; // (a weight that l counts stays below 2^98)
                    const float alpha = __builtin_amdgcn_exp2f((m - m_new) + (r - r_new));
                    l *= __builtin_amdgcn_exp2f(m - m_new);
                    m = m_new;
                    r = r_new;
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                        for (int v = 0; v < 16; ++v) ot[dt][v] *= alpha;
                }
                const float lr = (vexp - r) + vfrac + kKv8WeightExp;
                float nb = lr - m;
                if (special) { // next to a mask's -1e9 the scale's share would be rounded away: the difference first
#pragma unroll
                    for (int v = 0; v < 16; ++v) st[v] -= m;
                    nb = lr;
                }
                half8 ph[2], pl[2];
                float sum0 = 0.f, sum1 = 0.f;
                float minus1 = -1.0f; // opaque, so that e - h stays one mixed-precision FMA instead of a conversion and a subtraction
                asm volatile("" : "+s"(minus1));
#pragma unroll
                for (int v = 0; v < 16; v += 2) {
                    float2v e, rem;
                    e[0] = __builtin_amdgcn_exp2f(fmaf(st[v], cs, nb));
                    e[1] = __builtin_amdgcn_exp2f(fmaf(st[v + 1], cs, nb));
                    sum0 += e[0];
                    sum1 += e[1];
                    const half2v h = __builtin_convertvector(e, half2v);
                    rem[0] = fmaf((float)h[0], minus1, e[0]); // exact
                    rem[1] = fmaf((float)h[1], minus1, e[1]);
                    const half2v r = __builtin_convertvector(rem, half2v);
                    ph[v / 8][v % 8] = h[0]; ph[v / 8][v % 8 + 1] = h[1];
                    pl[v / 8][v % 8] = r[0]; pl[v / 8][v % 8 + 1] = r[1];
                }
                l = fmaf(sum0 + sum1, __builtin_amdgcn_exp2f(-lr), l);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    if (dt + 1 < NDT) v_stage((dt + 1) & 1, dt + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const half4 lo = vst[dt & 1][2 * u], hi = vst[dt & 1][2 * u + 1];
                        half8 va;
                        va[0] = lo[0]; va[1] = lo[1]; va[2] = lo[2]; va[3] = lo[3];
                        va[4] = hi[0]; va[5] = hi[1]; va[6] = hi[2]; va[7] = hi[3];
                        ot[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[u], ot[dt], 0, 0, 0);
                        ot[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[u], ot[dt], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            e0 = e1;
            e1 = e2;
            e2 = i + 3 < n ? __builtin_amdgcn_readfirstlane(list_entry(c0, i + 3)) : 0u;
        };
        for (int i = 0; i < n; i += 2) {
            tile_step(i, std::integral_constant<int, 0>{});
            if (i + 1 < n) tile_step(i + 1, std::integral_constant<int, 1>{});
        }
    }

    l += __shfl_xor(l, 32);
    const size_t slot = ((size_t)bh * QB + qb) * KS + split; // of the partials
    if (hf == 0 && q_row < tokens) {
        if (KS > 1) pp.part_ml[slot * pp.part_rows + wave * 32 + qi] = make_float2(m, l);
        else if (p.stats) p.stats[(size_t)bh * S + q_row] = make_float2(m, l);
    }
    // e^(..) sums to l, accumulators are in units of 2^r with weights times 2^7; a fully masked query: 0 / 0
    const float rl = __builtin_ldexpf(1.0f, (int)(r - kKv8WeightExp)) / (KS > 1 ? 1.0f : l);
    __syncthreads(); // every wave is done with the last tile
    float *so = reinterpret_cast<float *>(smem) + wave * 32 * LDO;
    const int q0 = qb * kPrefillQueriesPerBlock + wave * 32;
    float *dst0 = KS > 1 ? pp.part_o + (slot * pp.part_rows + wave * 32) * D : a.out + ((size_t)bh * S + q0) * D;
    constexpr int LPRW = HALF_D / 4, ROWS = 64 / LPRW;
#pragma unroll
    for (int pass = 0; pass < D / HALF_D; ++pass) {
#pragma unroll
        for (int dd = 0; dd < HALF_D / 32; ++dd) {
            const int dt = pass * (HALF_D / 32) + dd;
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<float4 *>(so + qi * LDO + 32 * dd + 8 * g4 + 4 * hf) =
                    make_float4(ot[dt][4 * g4 + 0] * rl, ot[dt][4 * g4 + 1] * rl, ot[dt][4 * g4 + 2] * rl, ot[dt][4 * g4 + 3] * rl);
        }
        wave_lds_sync();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const int r = r0 + lane / LPRW, c4 = lane % LPRW;
            float4 v = *reinterpret_cast<const float4 *>(so + r * LDO + 4 * c4);
            if (q0 + r >= tokens) v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (q0 + r < S) *reinterpret_cast<float4 *>(dst0 + (size_t)r * D + pass * HALF_D + 4 * c4) = v;
        }
        wave_lds_sync(); // the slice is rewritten by the next pass
    }
}

// Merges the key splits of every query: out = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(m_s - max m).  D/4 lanes per query;
// grid = ceil(B*H*S / (1024 / D)), block = 256.
template <int D>
__global__ __launch_bounds__(256) void kv8_prompt_merge_kernel(const Kv8PromptParams pp)
{
    constexpr int TPR = D / 4, ROWS = 256 / TPR; // (size_per_head 96: the last 16 threads own no query)
    const Kv8Params &p = pp.k;
    const int S = p.S, QB = (S + kPrefillQueriesPerBlock - 1) / kPrefillQueriesPerBlock, KS = pp.key_splits;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    if (threadIdx.x >= ROWS * TPR || row >= (int64_t)p.a.B * p.a.H * S) return;
    const int bh = (int)(row / S), q = (int)(row % S), t = threadIdx.x % TPR;
    const int tokens = kv8_prompt_tokens(p, bh / p.a.H);
    if (q >= tokens) {
        const float x = kv8_no_query(tokens);
        reinterpret_cast<float4 *>(p.a.out + (size_t)row * D)[t] = make_float4(x, x, x, x);
        return;
    }
    const size_t slot0 = ((size_t)bh * QB + q / kPrefillQueriesPerBlock) * KS, at = q % kPrefillQueriesPerBlock;
    float M = kMaxFloor * kLog2e;
    for (int s = 0; s < KS; ++s) M = fmaxf(M, pp.part_ml[(slot0 + s) * pp.part_rows + at].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < KS; ++s) {
        const size_t i = (slot0 + s) * pp.part_rows + at;
        const float2 ml = pp.part_ml[i];
        const float4 x = reinterpret_cast<const float4 *>(pp.part_o + i * D)[t];
        const float w = __builtin_amdgcn_exp2f(ml.x - M);
        l = fmaf(ml.y, w, l);
        o.x = fmaf(x.x, w, o.x); o.y = fmaf(x.y, w, o.y); o.z = fmaf(x.z, w, o.z); o.w = fmaf(x.w, w, o.w);
    }
    o.x /= l; o.y /= l; o.z /= l; o.w /= l;
    reinterpret_cast<float4 *>(p.a.out + (size_t)row * D)[t] = o;
    if (p.stats && t == 0) p.stats[row] = make_float2(M, l);
}

// Block weights of a prompt: weights[b,h,blk] (+)= sum over the last weight_queries queries and the block's rows of
// 2^(s' - m') / l, with the operands and statistics the attention kernel left.  Two products' worth of matrix instructions per
// query and key.  A wave keeps 64 keys in registers and walks the queries 32 at a time; the four waves of a workgroup are 4 / NQ
// groups of keys times NQ streams of queries.  STAGED (NQ = 1): the operands of a query block, 16 KB at D = 128, pass
// through LDS once for all four waves, the next block's on their way meanwhile; read by every wave for itself they are as
// much traffic at the L1 as the products take.  With NQ = 2 or 4 a workgroup is done sooner, where there are few of them.  The
// blocks that the mask leaves something of are listed first, with their classes, as in the attention kernel.
// grid = B*H * ceil(keys of the longest sequence / (256 / NQ)), heads fastest: under a causal mask the first keys' workgroups are
// the longest and start first, and an XCD keeps to its heads' operands; block = 256.  32 heads, 4096 queries, causal, all counted
// (two streams): 195-208 us (107 for the products at the library's rate; key groups fastest, classes behind each other 277).  Sums
// are formed in one order, so they are the same from run to run.
constexpr int kQueryListCap = 1024; // 32-query blocks per pass
template <int D, bool STAGED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 8)))
void kv8_prompt_weights_kernel(const Kv8PromptParams pp, int streams)
{
    constexpr int NC = D / 16, KT = 2, NS = NC / 2; // NS: 16-byte chunks of a query block per thread
    __shared__ half8 s_q[STAGED ? 2 : 1][STAGED ? 2 * NC * 64 : 1];
    __shared__ uint32_t s_list[kQueryListCap];
    __shared__ int s_cnt[4];
    __shared__ float s_sum[4][KT];
    const Kv8Params &p = pp.k;
    const Params &a = p.a;
    const int NQ = STAGED ? 1 : streams;
    const int S = p.S, P = a.start_pos, T = p.T, class_ld = (P + S + 31) / 32;
    const int keys = 256 / NQ;
    const int wg_key = blockIdx.x / (a.B * a.H) * keys, bh = blockIdx.x % (a.B * a.H);
    const int tokens = kv8_prompt_tokens(p, bh / a.H), ctx = P + tokens, ctx8 = ctx & ~(T - 1);
    if (tokens <= 0 || wg_key >= ctx) return; // (uniform)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, hf = lane >> 5;
    const int key0 = wg_key + wave / NQ * (32 * KT); // this wave's first key
    half8 ka[KT][NC]; // key key0 + 32 t + qi, elements 16c + 8hf ..
    float ks[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int k0 = key0 + 32 * t, row = k0 + qi;
        ks[t] = 1.f;
        if (k0 < ctx8) {
            ks[t] = p.k_scale[(size_t)bh * p.nblk + (k0 >> p.t_shift)];
            const int8_t *src = p.k8 + ((size_t)bh * a.L + row) * D + 8 * hf;
            uint2 x[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) x[c] = *reinterpret_cast<const uint2 *>(src + 16 * c);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                half2v h[4];
                widen4(x[c].x, h[0], h[1]);
                widen4(x[c].y, h[2], h[3]);
#pragma unroll
                for (int i = 0; i < 8; ++i) ka[t][c][i] = h[i / 2][i % 2];
            }
        } else { // the tail, zeros behind it
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                ka[t][c] = half8{0, 0, 0, 0, 0, 0, 0, 0};
                if (row < ctx) ka[t][c] = *reinterpret_cast<const half8 *>(p.k_tail + ((size_t)bh * T + (row - ctx8)) * D + 16 * c + 8 * hf);
            }
        }
    }
    const int first_query = tokens - p.weight_queries, first_block = first_kept_block(p, tokens), blocks = (tokens + 31) / 32 - first_block;
    // The 32-query blocks [b0, b1) that some key of this workgroup counts for: (block - b0) << 16 | two bits of class per key tile.
    auto build_list = [&](int b0, int b1) __attribute__((always_inline)) -> int {
        int count = 0;
        for (int base = b0; base < b1; base += 256) {
            const int block = base + tid, q0 = (first_block + block) * 32;
            uint32_t cls = 0u;
            if (block < b1) {
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    if (t * 32 >= keys || wg_key + 32 * t >= ctx) continue;
                    const uint32_t c = a.attn_mask ? prompt_class_word(pp.f, q0 / kPrefillQueriesPerBlock, wg_key / 32 + t, class_ld) >> (8 * (q0 / 32 % 4)) : kTileZero;
                    cls |= (c & 3u) << (2 * t);
                }
            }
            const unsigned long long bal = __ballot(cls != 0u);
            if (lane == 0) s_cnt[wave] = __popcll(bal);
            __syncthreads();
            int at = count + __popcll(bal & ((1ull << lane) - 1ull));
            for (int w = 0; w < wave; ++w) at += s_cnt[w];
            if (cls != 0u) s_list[at] = (uint32_t)(block - b0) << 16 | cls;
            count += s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3];
            __syncthreads();
        }
        return count;
    };
    float sum[KT] = {0.f, 0.f};
    for (int b0 = 0; b0 < blocks; b0 += kQueryListCap) {
        const int n = build_list(b0, min(b0 + kQueryListCap, blocks));
        auto operands_at = [&](uint32_t entry) __attribute__((always_inline)) -> const half8 * {
            return pp.q_pairs + ((size_t)bh * pp.kept_blocks + b0 + (entry >> 16)) * (2 * NC * 64);
        };
        half8 stage[NS];
        float2 ml_next;
        float factor_next;
        auto fetch = [&](int i) __attribute__((always_inline)) { // of list entry i: statistics and, staged, this thread's chunks
            const uint32_t entry = __builtin_amdgcn_readfirstlane(s_list[i]);
            const int block = b0 + (int)(entry >> 16);
            if constexpr (STAGED) {
                const half8 *src = operands_at(entry) + tid;
#pragma unroll
                for (int j = 0; j < NS; ++j) stage[j] = src[j * 256];
            }
            ml_next = p.stats[(size_t)bh * S + min((first_block + block) * 32 + qi, S - 1)];
            factor_next = pp.q_factor[((size_t)bh * pp.kept_blocks + block) * 32 + qi];
        };
        int i = wave % NQ;
        if (i < n) fetch(i);
        for (int parity = 0; i < n; i += NQ, parity ^= 1) {
            const uint32_t entry = __builtin_amdgcn_readfirstlane(s_list[i]);
            const int q = (first_block + b0 + (int)(entry >> 16)) * 32 + qi, q_in = min(q, S - 1);
            const float2 ml = ml_next;
            const float factor = factor_next;
            if constexpr (STAGED) {
#pragma unroll
                for (int j = 0; j < NS; ++j) s_q[parity][tid + j * 256] = stage[j];
                __syncthreads(); // the block is there; everyone is done with the one before the last
            }
            half8 direct[STAGED ? 1 : 2 * NC];
            if constexpr (!STAGED) {
                const half8 *src = operands_at(entry) + lane;
#pragma unroll
                for (int c = 0; c < 2 * NC; ++c) direct[c] = src[c * 64];
            }
            if (i + NQ < n) fetch(i + NQ);
            uint32_t cls[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) cls[t] = (entry >> (2 * (wave / NQ * KT + t))) & 3u;
            if (cls[0] == kTileSkip && cls[1] == kTileSkip) continue;
            floatx16 st[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int v = 0; v < 16; ++v) st[t][v] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const half8 hi = STAGED ? s_q[STAGED ? parity : 0][STAGED ? c * 64 + lane : 0] : direct[STAGED ? 0 : c];
                const half8 lo = STAGED ? s_q[STAGED ? parity : 0][STAGED ? (NC + c) * 64 + lane : 0] : direct[STAGED ? 0 : NC + c];
#pragma unroll
                for (int t = 0; t < KT; ++t) st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[t][c], lo, st[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < KT; ++t) st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[t][c], hi, st[t], 0, 0, 0);
            }
            // a query of the call that counts, and that saw a key
            const float rl = q >= first_query && q < tokens && ml.y > 0.f ? 1.0f / ml.y : 0.f;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                if (cls[t] == kTileSkip) continue; // uniform
                const int k0 = key0 + 32 * t;
                const float cs = factor * ks[t];
                if (cls[t] >= kTileMixed || k0 + 32 > ctx) { // uniform
                    const float *mrow = a.attn_mask + (size_t)(P + q_in) * a.mask_ld;
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const int key = 8 * (v / 4) + 4 * hf + (v % 4);
                        float x = st[t][v] * cs;
                        if (cls[t] == kTileMixed) x = fmaf(mrow[min(k0 + key, ctx - 1)], kLog2e, x);
                        st[t][v] = (cls[t] == kTileDiag && key > qi) || k0 + key >= ctx ? -__builtin_inff() : x - ml.x;
                    }
                } else {
#pragma unroll
                    for (int v = 0; v < 16; ++v) st[t][v] = fmaf(st[t][v], cs, -ml.x);
                }
                float part = 0.f;
#pragma unroll
                for (int v = 0; v < 16; ++v) part += __builtin_amdgcn_exp2f(st[t][v]);
                if (rl > 0.f) sum[t] = fmaf(part, rl, sum[t]);
            }
        }
        if (b0 + kQueryListCap < blocks) __syncthreads(); // the list and the buffers are written again
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        sum[t] = wave_sum(sum[t]);
        if (lane == 0) s_sum[wave][t] = sum[t];
    }
    __syncthreads();
    const int row0 = wg_key + tid * T; // one thread per block of this workgroup's keys (whole blocks: T <= 256 / NQ)
    if (tid < keys / T && row0 < ctx) {
        float w = 0.f;
        for (int t = tid * T / 32; t < (tid + 1) * T / 32; ++t) // 32-key tile t: group t / KT
            for (int k = 0; k < NQ; ++k) w += s_sum[t / KT * NQ + k][t % KT];
        float *dst = p.weights + (size_t)bh * p.nblk + (row0 >> p.t_shift);
        *dst = row0 >= P ? w : *dst + w;
    }
}

} // namespace flattn
