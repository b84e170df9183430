// C ABI of the 8-bit key/value cache (see include/fl_decode_attn.h): validation, planning and dispatch.  Enqueue-only, as
// fl_decode_attn.hip: no allocation, no synchronisation, nothing remembered about the caller.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/fl_decode_attn.h"
#include "capi_common.hpp"
#include "kv8_kernels.hpp"
#include "kv8_prefill_kernels.hpp"

namespace {

using namespace flhost;
using flattn::Kv8EvictParams;
using flattn::Kv8Params;
using flattn::Kv8PromptParams;

constexpr size_t kCacheMinBytes = offsetof(fl_kv8_cache, weights) + sizeof(void *);
constexpr size_t kEvictMinBytes = offsetof(fl_kv8_evict_args, rows_out) + sizeof(void *);
constexpr int kChunkRows = 128; // splits are multiples of it, hence of every block length

bool block_len_ok(int T) { return T == 32 || T == 64 || T == 128; }
int log2_of(int T) { return T == 32 ? 5 : (T == 64 ? 6 : 7); }

int validate_block(const fl_attn_desc *d, int T)
{
    return block_len_ok(T) && d->total_len % T == 0 ? FL_ATTN_OK : FL_ATTN_ERR_SHAPE;
}

int import_cache(const fl_attn_desc *d, const fl_kv8_cache *in, fl_kv8_cache *c)
{
    int st = import_struct(in, c, kCacheMinBytes);
    if (st != FL_ATTN_OK) return st;
    st = validate_block(d, c->block_len);
    if (st != FL_ATTN_OK) return st;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail) return FL_ATTN_ERR_NULL_POINTER;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_tail) || !aligned16(c->v_tail)) return FL_ATTN_ERR_ALIGNMENT;
    for (const void *f : {(const void *)c->k_scale, (const void *)c->v_scale, (const void *)c->weights})
        if ((reinterpret_cast<uintptr_t>(f) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT;
    return FL_ATTN_OK;
}

int granule_rows(int D) // Kv8Geometry<D>::GR
{
    const int wt = 4 * 64 / flattn::lanes_per_row(D / 16);
    return wt < 32 ? wt : 32;
}

// ---- launch planning of the decode step: `nsplit` workgroups per (b,h), all but the last with a multiple of kChunkRows rows of
// the complete blocks, the last with the open block (its rows are few, but the append comes first); a context that is
// not split is one workgroup.
constexpr size_t kRaggedChunkBytes = 256 * 1024;

int byte_splits(const fl_attn_desc *d, int ctx, bool ragged)
{
    const int64_t bh = (int64_t)d->batch_size * d->head_num;
    int64_t n = (device_cus() + bh - 1) / bh;
    if (ctx <= 2 * kChunkRows) n = 1;
    if (ragged) { // work per (b,h) varies
        const int64_t by_bytes = ((int64_t)ctx * 2 * d->size_per_head + kRaggedChunkBytes - 1) / (int64_t)kRaggedChunkBytes;
        if (by_bytes > n) n = by_bytes;
    }
    if (d->nsplit > 0) n = d->nsplit;
    const int64_t most = ((int64_t)ctx + kChunkRows - 1) / kChunkRows;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : (n > kMaxSplits - 1 ? kMaxSplits - 1 : n));
}

int split_cap(const fl_attn_desc *d) { return byte_splits(d, d->total_len, true) + 1; }

void make_plan(const fl_attn_desc *d, int ctx, bool ragged, fl_attn_plan *plan)
{
    const int n = byte_splits(d, ctx, ragged);
    plan->chunk_rows = ((ctx + n - 1) / n + kChunkRows - 1) / kChunkRows * kChunkRows;
    plan->nsplit = n == 1 ? 1 : (ctx + plan->chunk_rows - 1) / plan->chunk_rows + 1;
    plan->threads = flattn::kKv8Waves * 64;
    plan->two_pass = plan->nsplit <= 1 ? 0 : ((int64_t)plan->nsplit * d->batch_size * d->head_num <= 4 * (int64_t)device_cus() ? 2 : 1);
}

// Workspace: [arrivals B*H] [float output B*H*S*D] [part_o] [part_m] [part_l] [granules] [mask tile classes], and for the
// block weights of a prompt [statistics B*H*S] [query operands] [query factors]; 256-byte sections.
struct Layout {
    size_t arrivals, tmp_out, part_o, part_m, part_l, granules, tile_class, stats, q_pairs, q_factor, prompt_o, prompt_ml, total;
};

constexpr int kPromptWorkgroups = 512, kPromptMinTiles = 4;
int partial_rows(int S) { return S < flattn::kPrefillQueriesPerBlock ? S : flattn::kPrefillQueriesPerBlock; }

Layout layout(const fl_attn_desc *d, int S)
{
    const size_t bh = (size_t)d->batch_size * d->head_num, D = d->size_per_head, slots = bh * (size_t)split_cap(d);
    const size_t qblocks = ((size_t)S + flattn::kPrefillQueriesPerBlock - 1) / flattn::kPrefillQueriesPerBlock;
    const size_t ktiles = ((size_t)d->total_len + flattn::kPrefillKeysPerStep - 1) / flattn::kPrefillKeysPerStep;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += align_up(bytes, 256); return here; };
    Layout w;
    w.arrivals = take(bh * 4);
    w.tmp_out = take(bh * (size_t)S * D * 4);
    w.part_o = take(slots * D * 4);
    w.part_m = take(slots * 4);
    w.part_l = take(slots * 4);
    w.granules = take(bh * (size_t)(d->total_len / granule_rows(d->size_per_head)) * 8);
    w.tile_class = take(qblocks * ktiles * 4);
    const size_t S32 = ((size_t)S + 31) / 32 * 32;
    w.stats = take(bh * S32 * 8);
    w.q_pairs = take(D <= 128 ? bh * S32 * D * 4 : 0);
    w.q_factor = take(bh * S32 * 4);
    // key splits of a prompt: at most kPromptWorkgroups partials (for this and for every shorter prompt) of up to 128 queries
    const size_t rows = D <= 128 && bh * 2 <= kPromptWorkgroups ? kPromptWorkgroups * (size_t)partial_rows(S) : 0;
    w.prompt_o = take(rows * D * 4);
    w.prompt_ml = take(rows * 8);
    w.total = at;
    return w;
}

// Workgroups that share the keys of a (128-query block, head) of a prompt.  One workgroup walks its tiles at about 1 us each,
// however few others there are, so a short piece behind a long context is bound by that walk; where the query blocks leave
// the compute units' two workgroup slots empty, the keys are split, down to four tiles each, and a second launch merges.
// Measured, whole call without / with the split, us (D = 128): 16 queries after 4000, 4 heads 166 / 36, 32 heads 171 / 39; 128 after
// 1024, 8 heads 61 / 30; B=3, 5 heads (D = 96), 333 after 77 27.9 / 26.1; 512 queries, 32 heads 39.5 / 41.3.  Eight tiles
// each are as good at 4000 rows and 2-4 us worse at 600-1500, two are 4-8 us worse; 1024 workgroups 55 at the second shape.
int prompt_key_splits(const fl_attn_desc *d, int ctx, int S)
{
    if (d->size_per_head > 128) return 1;
    const int64_t blocks = (int64_t)d->batch_size * d->head_num * ((S + flattn::kPrefillQueriesPerBlock - 1) / flattn::kPrefillQueriesPerBlock);
    const int64_t tiles = (ctx + flattn::kPrefillKeysPerStep - 1) / flattn::kPrefillKeysPerStep;
    int64_t n = kPromptWorkgroups / blocks;
    if (n > tiles / kPromptMinTiles) n = tiles / kPromptMinTiles;
    return (int)(n < 1 ? 1 : n);
}

int check_workspace(const void *ws, size_t bytes, const Layout &w)
{
    return ws && bytes >= w.total && (reinterpret_cast<uintptr_t>(ws) & 255u) == 0 ? FL_ATTN_OK : FL_ATTN_ERR_WORKSPACE;
}

// What both phases ask of io.
int check_io(const fl_attn_io *io)
{
    if (!io->q || !io->k_new || !io->v_new || !io->freq_cis) return FL_ATTN_ERR_NULL_POINTER;
    const bool quant = io->out_int8 != nullptr, i32 = io->qkv_inp_scale != nullptr;
    if (!io->out && !quant) return FL_ATTN_ERR_NULL_POINTER;
    if (quant && !io->out_scale) return FL_ATTN_ERR_NULL_POINTER;
    if (quant && (reinterpret_cast<uintptr_t>(io->out_int8) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT; // written four at a time
    if (i32 && (!io->q_weight_scale || !io->k_weight_scale || !io->v_weight_scale)) return FL_ATTN_ERR_NULL_POINTER;
    if (!i32 && (io->q_weight_scale || io->k_weight_scale || io->v_weight_scale)) return FL_ATTN_ERR_ARGUMENT;
    if (!aligned16(io->q) || !aligned16(io->k_new) || !aligned16(io->v_new) || !aligned16(io->freq_cis) || !aligned16(io->out) ||
        (i32 && (!aligned16(io->q_weight_scale) || !aligned16(io->k_weight_scale) || !aligned16(io->v_weight_scale))))
        return FL_ATTN_ERR_ALIGNMENT;
    if (io->rope_row < FL_ATTN_ROPE_AT_POSITION) return FL_ATTN_ERR_POSITION;
    return FL_ATTN_OK;
}

Kv8Params make_params(const fl_attn_desc *d, const fl_kv8_cache *c, const fl_attn_io *io)
{
    Kv8Params p{};
    p.a.q = io->q; p.a.k_new = io->k_new; p.a.v_new = io->v_new;
    p.a.freq_cis = io->freq_cis; p.a.attn_mask = io->attn_mask; p.a.mask_ld = io->mask_ld;
    p.a.inp_scale = io->qkv_inp_scale; p.a.wq_scale = io->q_weight_scale; p.a.wk_scale = io->k_weight_scale; p.a.wv_scale = io->v_weight_scale;
    p.a.start_pos = io->start_pos; p.a.rope_row = io->rope_row;
    p.in_kind = io->qkv_inp_scale ? flattn::kInI32 : (d->dtype == FL_ATTN_F16 ? flattn::kInF16 : flattn::kInF32);
    p.a.B = d->batch_size; p.a.H = d->head_num; p.a.L = d->total_len;
    p.a.scale = d->softmax_scale > 0.f ? d->softmax_scale : 1.0f / sqrtf((float)d->size_per_head);
    p.a.log2_domain = 1;
    p.k8 = c->k; p.v8 = c->v; p.k_scale = c->k_scale; p.v_scale = c->v_scale;
    p.k_tail = static_cast<_Float16 *>(c->k_tail); p.v_tail = static_cast<_Float16 *>(c->v_tail);
    p.weights = c->weights;
    p.T = c->block_len; p.t_shift = log2_of(c->block_len); p.nblk = d->total_len / c->block_len;
    p.S = 1;
    return p;
}

template <int D>
hipError_t launch_decode(const Kv8Params &p, const fl_attn_plan &plan, hipStream_t stream)
{
    const unsigned bh = (unsigned)(p.a.B * p.a.H);
    const dim3 grid((unsigned)plan.nsplit * bh), block(flattn::kKv8Waves * 64);
    hipError_t e = p.a.attn_mask ? launch(flattn::kv8_attn_kernel<D, true, false>, grid, block, stream, p)
                                 : launch(flattn::kv8_attn_kernel<D, false, false>, grid, block, stream, p);
    if (e != hipSuccess || p.a.direct || p.a.arrivals) return e;
    return launch(flattn::kv8_combine_kernel<D>, dim3(bh), dim3(flattn::kCombineThreads), stream, p);
}

template <int D>
hipError_t launch_append(const Kv8Params &p, hipStream_t stream)
{
    const int n = (p.a.start_pos + p.S) / p.T - p.a.start_pos / p.T;
    const dim3 grid((unsigned)(p.a.B * p.a.H * 2 * (n > 0 ? n : 1))), block(256);
    if (p.T == 32) return launch(flattn::kv8_append_kernel<D, 32>, grid, block, stream, p);
    if (p.T == 64) return launch(flattn::kv8_append_kernel<D, 64>, grid, block, stream, p);
    return launch(flattn::kv8_append_kernel<D, 128>, grid, block, stream, p);
}

template <int D>
hipError_t launch_prompt(const Kv8PromptParams &pp, hipStream_t stream)
{
    const Kv8Params &p = pp.k;
    hipError_t e = launch_append<D>(p, stream);
    if (e != hipSuccess) return e;
    const unsigned bh = (unsigned)(p.a.B * p.a.H);
    if constexpr (D > 128) { // the matrix-core kernel's state no longer fits: one workgroup per query
        const dim3 grid((unsigned)p.S * bh), block(flattn::kKv8Waves * 64);
        if (p.a.attn_mask) return launch(flattn::kv8_attn_kernel<D, true, true>, grid, block, stream, p);
        return launch(flattn::kv8_attn_kernel<D, false, true>, grid, block, stream, p);
    } else {
        const unsigned qblocks = (unsigned)((p.S + flattn::kPrefillQueriesPerBlock - 1) / flattn::kPrefillQueriesPerBlock);
        if (p.a.attn_mask && !pp.f.class_table && pp.f.tile_class) { // no table of the whole mask at hand: classify the rows of this call
            const int ktiles = (p.a.start_pos + p.S + flattn::kPrefillKeysPerStep - 1) / flattn::kPrefillKeysPerStep;
            e = launch(flattn::prefill_mask_classify_kernel, dim3((unsigned)ktiles, qblocks), dim3(256), stream, pp.f, ktiles);
            if (e != hipSuccess) return e;
        }
        const dim3 grid(qblocks * bh * (unsigned)pp.key_splits), block(256);
        e = p.a.attn_mask ? launch(flattn::kv8_prefill_attn_kernel<D, true>, grid, block, stream, pp)
                          : launch(flattn::kv8_prefill_attn_kernel<D, false>, grid, block, stream, pp);
        if (e != hipSuccess) return e;
        if (pp.key_splits > 1) {
            const int64_t rows = (int64_t)bh * p.S;
            constexpr int per = 256 / (D / 4);
            e = launch(flattn::kv8_prompt_merge_kernel<D>, dim3((unsigned)((rows + per - 1) / per)), block, stream, pp);
            if (e != hipSuccess) return e;
        }
        if (!p.stats) return e;
        // Query streams per workgroup of the block weights (see the kernel).  More streams, more and shorter workgroups, but each
        // reads the operands for fewer keys: split until there are four workgroups per compute unit (under a causal mask the
        // first keys' workgroups see every query, and with two per unit they finish last), or one where there are only a few
        // query blocks per stream; a workgroup's 256 / NQ keys are whole blocks.  The whole call, in us, for NQ = 1 / 2 / 4, D = 128:
        //   32 heads, 4096 queries, all counted  512 / 481 / 473     the last 64   315 / 321 / 334
        //   B=8, 32 heads, 1024, all             326 / 345 / 393     the last 64   234 / 246 / 270
        //   8 heads, 2048, all                   161 / 104 /  87     B=3, 5 heads (D = 96), 333, all   47 / 40 / 37
        const int ctx = p.a.start_pos + p.S;
        int NQ = 1;
        while (NQ < 4 && 2 * NQ * p.T <= 256 && NQ < pp.kept_blocks &&
               (int64_t)((ctx + 256 / NQ - 1) / (256 / NQ)) * bh < (4 * NQ < pp.kept_blocks ? 4 : 1) * (int64_t)device_cus())
            NQ *= 2;
        const dim3 weights_grid((unsigned)((ctx + 256 / NQ - 1) / (256 / NQ)) * bh);
        return NQ == 1 ? launch(flattn::kv8_prompt_weights_kernel<D, true>, weights_grid, block, stream, pp, 1)
                       : launch(flattn::kv8_prompt_weights_kernel<D, false>, weights_grid, block, stream, pp, NQ);
    }
}

#define KV8_BY_HEAD_SIZE(D, F, ...)                    \
    switch (D) {                                       \
    case 32: return F<32>(__VA_ARGS__);                \
    case 64: return F<64>(__VA_ARGS__);                \
    case 96: return F<96>(__VA_ARGS__);                \
    case 128: return F<128>(__VA_ARGS__);              \
    case 256: return F<256>(__VA_ARGS__);              \
    case 512: return F<512>(__VA_ARGS__);              \
    case 1024: return F<1024>(__VA_ARGS__);            \
    default: return hipErrorInvalidValue;              \
    }

hipError_t dispatch_decode(int D, const Kv8Params &p, const fl_attn_plan &plan, hipStream_t s) { KV8_BY_HEAD_SIZE(D, launch_decode, p, plan, s) }
hipError_t dispatch_prompt(int D, const Kv8PromptParams &p, hipStream_t s) { KV8_BY_HEAD_SIZE(D, launch_prompt, p, s) }
#undef KV8_BY_HEAD_SIZE

__global__ static void kv8_fill_zero_kernel(int32_t *dst, int64_t n)
{
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i < n) dst[i] = 0;
}

constexpr int64_t kEvictOneLaunchBytes = 128 * 1024; // kept rows of one (b,h), K and V

bool overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

} // namespace

extern "C" {

int fl_kv8_cache_bytes(const fl_attn_desc *desc, int32_t block_len, size_t *rows_bytes, size_t *scale_bytes, size_t *tail_bytes)
{
    if (!rows_bytes || !scale_bytes || !tail_bytes) return FL_ATTN_ERR_NULL_POINTER;
    fl_attn_desc copy;
    int st = import_desc(&desc, &copy);
    if (st == FL_ATTN_OK) st = validate_block(desc, block_len);
    if (st != FL_ATTN_OK) return st;
    const size_t bh = (size_t)desc->batch_size * desc->head_num, L = desc->total_len, D = desc->size_per_head;
    *rows_bytes = bh * L * D;
    *scale_bytes = bh * (L / block_len) * sizeof(float);
    *tail_bytes = bh * block_len * D * 2;
    return FL_ATTN_OK;
}

int fl_kv8_workspace_bytes(const fl_attn_desc *desc, int32_t block_len, int32_t seq_len, size_t *bytes)
{
    if (!bytes) return FL_ATTN_ERR_NULL_POINTER;
    fl_attn_desc copy;
    int st = import_desc(&desc, &copy);
    if (st == FL_ATTN_OK) st = validate_block(desc, block_len);
    if (st != FL_ATTN_OK) return st;
    if (seq_len < 1 || seq_len > desc->total_len) return FL_ATTN_ERR_POSITION;
    *bytes = layout(desc, seq_len).total;
    return FL_ATTN_OK;
}

int fl_kv8_workspace_init(const fl_attn_desc *desc, int32_t block_len, int32_t seq_len, void *workspace, size_t workspace_bytes, void *hip_stream)
{
    size_t need;
    int st = fl_kv8_workspace_bytes(desc, block_len, seq_len, &need);
    if (st != FL_ATTN_OK) return st;
    fl_attn_desc copy;
    import_desc(&desc, &copy);
    const Layout w = layout(desc, seq_len);
    st = check_workspace(workspace, workspace_bytes, w);
    if (st != FL_ATTN_OK) return st;
    const int64_t n = (int64_t)desc->batch_size * desc->head_num;
    // a fill kernel, not a memset: memset nodes are the one thing a caller cannot safely capture in a HIP graph
    if (!check_hip(launch(kv8_fill_zero_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), static_cast<hipStream_t>(hip_stream),
                          reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + w.arrivals), n)))
        return FL_ATTN_ERR_HIP;
    return FL_ATTN_OK;
}

int fl_kv8_decode_forward(const fl_attn_desc *desc, const fl_kv8_cache *cache, const fl_attn_io *io_in, const int32_t *rope_row_per_seq, int32_t rope_table_rows,
                          void *hip_stream)
{
    fl_attn_desc desc_copy;
    int st = import_desc(&desc, &desc_copy);
    if (st != FL_ATTN_OK) return st;
    fl_kv8_cache c;
    st = import_cache(desc, cache, &c);
    if (st != FL_ATTN_OK) return st;
    fl_attn_io io;
    st = import_struct(io_in, &io, kIoMinBytes);
    if (st != FL_ATTN_OK) return st;
    st = check_io(&io);
    if (st != FL_ATTN_OK) return st;
    if ((io.flags & ~FL_ATTN_IO_WORKSPACE_READY) != 0) return FL_ATTN_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(rope_row_per_seq) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT;
    if (rope_row_per_seq && rope_table_rows < 1) return FL_ATTN_ERR_POSITION;
    const int L = desc->total_len, D = desc->size_per_head;
    const bool ragged = io.start_pos_per_seq != nullptr;
    int max_pos = io.start_pos;
    if (ragged) max_pos = io.max_start_pos < 0 ? L - 1 : io.max_start_pos;
    if (max_pos < 0 || max_pos >= L) return FL_ATTN_ERR_POSITION;
    if (io.attn_mask && (io.mask_ld < 0 || (io.mask_ld != 0 && io.mask_ld < (int64_t)max_pos + 1))) return FL_ATTN_ERR_ARGUMENT;

    fl_attn_plan plan;
    make_plan(desc, max_pos + 1, ragged, &plan);
    const int cap = split_cap(desc);
    if (plan.nsplit > cap) return FL_ATTN_ERR_ARGUMENT;
    const Layout w = layout(desc, 1);
    const bool direct = plan.nsplit == 1;
    if (!direct || c.weights || !io.out) {
        st = check_workspace(io.workspace, io.workspace_bytes, w);
        if (st != FL_ATTN_OK) return st;
    }
    char *ws = static_cast<char *>(io.workspace);
    Kv8Params p = make_params(desc, &c, &io);
    p.a.pos_per_seq = io.start_pos_per_seq;
    p.rope_rows = rope_row_per_seq;
    p.table_rows = rope_table_rows;
    p.a.out = io.out ? io.out : reinterpret_cast<float *>(ws + w.tmp_out);
    p.a.max_pos = max_pos; p.a.chunk = plan.chunk_rows; p.a.split_cap = cap; p.a.direct = direct;
    if (!direct) {
        p.a.part_o = reinterpret_cast<float *>(ws + w.part_o);
        p.a.part_m = reinterpret_cast<float *>(ws + w.part_m);
        p.a.part_l = reinterpret_cast<float *>(ws + w.part_l);
        if (plan.two_pass == 2 && (io.flags & FL_ATTN_IO_WORKSPACE_READY)) p.a.arrivals = reinterpret_cast<int32_t *>(ws + w.arrivals);
    }
    if (c.weights) p.granules = reinterpret_cast<float2 *>(ws + w.granules);
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if (!check_hip(dispatch_decode(D, p, plan, stream))) return FL_ATTN_ERR_HIP;
    if (io.out_int8 && !check_hip(launch(flattn::attn_quantize_transpose_kernel, dim3(desc->batch_size), dim3(flattn::kQuantThreads), stream,
                                         p.a.out, io.out_int8, io.out_scale, desc->head_num, 1, D)))
        return FL_ATTN_ERR_HIP;
    return FL_ATTN_OK;
}

int fl_kv8_prefill_forward(const fl_attn_desc *desc, const fl_kv8_cache *cache, const fl_attn_io *io_in, int32_t seq_len, const int32_t *seq_len_per_seq,
                           int32_t weight_queries, void *hip_stream)
{
    fl_attn_desc desc_copy;
    int st = import_desc(&desc, &desc_copy);
    if (st != FL_ATTN_OK) return st;
    fl_kv8_cache c;
    st = import_cache(desc, cache, &c);
    if (st != FL_ATTN_OK) return st;
    fl_attn_io io;
    st = import_struct(io_in, &io, kIoMinBytes);
    if (st != FL_ATTN_OK) return st;
    st = check_io(&io);
    if (st != FL_ATTN_OK) return st;
    if ((io.flags & ~FL_ATTN_IO_WORKSPACE_READY) != 0 || io.start_pos_per_seq || weight_queries < 0) return FL_ATTN_ERR_ARGUMENT; // all start at one position
    if ((reinterpret_cast<uintptr_t>(seq_len_per_seq) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT;
    const int L = desc->total_len, D = desc->size_per_head;
    if (seq_len < 1 || io.start_pos < 0 || (int64_t)io.start_pos + seq_len > L) return FL_ATTN_ERR_POSITION;
    if (io.attn_mask && (io.mask_ld < 0 || (io.mask_ld != 0 && io.mask_ld < (int64_t)io.start_pos + seq_len))) return FL_ATTN_ERR_ARGUMENT;
    if (c.weights && D > 128) return FL_ATTN_ERR_HEAD_DIM;
    // A launch has fewer than 2^32 threads: two workgroups per head and block that is filled, one per query and head where the head
    // size is beyond 128, one per token for INT8 output; the mask's classes are a two-dimensional grid.
    const int64_t queries = (int64_t)desc->batch_size * desc->head_num * seq_len;
    const int64_t filled = (io.start_pos + seq_len) / c.block_len - io.start_pos / c.block_len;
    if (queries > (int64_t)INT32_MAX || (int64_t)desc->batch_size * desc->head_num * 2 * filled > (int64_t)(UINT32_MAX / 256) ||
        (D > 128 && queries > (int64_t)(UINT32_MAX / (flattn::kKv8Waves * 64))) ||
        (io.out_int8 && (int64_t)desc->batch_size * seq_len > (int64_t)(UINT32_MAX / flattn::kQuantThreads)) ||
        seq_len > 65535 * flattn::kPrefillQueriesPerBlock)
        return FL_ATTN_ERR_SHAPE;
    const Layout w = layout(desc, seq_len);
    st = check_workspace(io.workspace, io.workspace_bytes, w);
    if (st != FL_ATTN_OK) return st;
    char *ws = static_cast<char *>(io.workspace);
    Kv8Params p = make_params(desc, &c, &io);
    p.a.out = io.out ? io.out : reinterpret_cast<float *>(ws + w.tmp_out);
    p.S = seq_len;
    p.tokens_per_seq = seq_len_per_seq;
    Kv8PromptParams pp{};
    flattn::PrefillParams &f = pp.f;
    f.attn_mask = io.attn_mask; f.mask_ld = io.mask_ld;
    if (io.start_pos + seq_len > flattn::kUnclassifiedKeys) f.tile_class = reinterpret_cast<uint32_t *>(ws + w.tile_class);
    f.B = desc->batch_size; f.H = desc->head_num; f.L = L; f.S = seq_len; f.start_pos = io.start_pos;
    if (io.mask_tile_classes && io.attn_mask && io.mask_ld >= L && io.start_pos % 32 == 0) {
        if ((reinterpret_cast<uintptr_t>(io.mask_tile_classes) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT; // read a word at a time
        f.class_table = static_cast<const uint8_t *>(io.mask_tile_classes);
        f.class_ld = (int32_t)class_table_ld(L);
    }
    if (c.weights) {
        p.stats = reinterpret_cast<float2 *>(ws + w.stats);
        p.weight_queries = weight_queries > 0 && weight_queries < seq_len ? weight_queries : seq_len;
        pp.q_pairs = reinterpret_cast<flattn::half8 *>(ws + w.q_pairs);
        pp.q_factor = reinterpret_cast<float *>(ws + w.q_factor);
        // the last W queries lie in (W + 31) / 32 blocks where the sequence's end is a block's, else in one more
        const int blocks = (seq_len + 31) / 32, spanned = seq_len_per_seq ? (p.weight_queries + 31) / 32 + 1 : blocks - (seq_len - p.weight_queries) / 32;
        pp.kept_blocks = spanned < blocks ? spanned : blocks;
    }
    pp.key_splits = prompt_key_splits(desc, io.start_pos + seq_len, seq_len);
    if (pp.key_splits > 1) {
        pp.part_o = reinterpret_cast<float *>(ws + w.prompt_o);
        pp.part_ml = reinterpret_cast<float2 *>(ws + w.prompt_ml);
        pp.part_rows = partial_rows(seq_len);
    }
    pp.k = p;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if (!check_hip(dispatch_prompt(D, pp, stream))) return FL_ATTN_ERR_HIP;
    if (io.out_int8 && !check_hip(launch(flattn::attn_quantize_transpose_kernel, dim3((unsigned)(desc->batch_size * seq_len)), dim3(flattn::kQuantThreads),
                                         stream, p.a.out, io.out_int8, io.out_scale, desc->head_num, seq_len, D)))
        return FL_ATTN_ERR_HIP;
    return FL_ATTN_OK;
}

int fl_kv8_read(const fl_attn_desc *desc, const fl_kv8_cache *cache, int32_t rows, const int32_t *rows_per_seq, void *k_out, void *v_out, void *hip_stream)
{
    fl_attn_desc desc_copy;
    int st = import_desc(&desc, &desc_copy);
    if (st != FL_ATTN_OK) return st;
    fl_kv8_cache c;
    st = import_cache(desc, cache, &c);
    if (st != FL_ATTN_OK) return st;
    if (!k_out || !v_out) return FL_ATTN_ERR_NULL_POINTER;
    if (!aligned16(k_out) || !aligned16(v_out) || (reinterpret_cast<uintptr_t>(rows_per_seq) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT;
    if (rows < 1 || rows > desc->total_len) return FL_ATTN_ERR_POSITION;
    const flattn::Kv8ReadParams p = {c.k, c.v, c.k_scale, c.v_scale, static_cast<const _Float16 *>(c.k_tail), static_cast<const _Float16 *>(c.v_tail),
                                     rows_per_seq, desc->head_num, desc->total_len, c.block_len, log2_of(c.block_len)};
    const int D = desc->size_per_head, vec = desc->dtype == FL_ATTN_F16 ? 8 : 4;
    const int64_t groups = ((int64_t)rows * (D / vec) + 1023) / 1024, grid = groups * 2 * desc->batch_size * desc->head_num;
    if (grid > INT32_MAX / 128) return FL_ATTN_ERR_SHAPE; // 2^32 threads a launch
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = desc->dtype == FL_ATTN_F16
                             ? launch(flattn::kv8_read_kernel<_Float16>, dim3((unsigned)grid), dim3(256), stream, p, static_cast<_Float16 *>(k_out),
                                      static_cast<_Float16 *>(v_out), rows, D, (int)groups)
                             : launch(flattn::kv8_read_kernel<float>, dim3((unsigned)grid), dim3(256), stream, p, static_cast<float *>(k_out),
                                      static_cast<float *>(v_out), rows, D, (int)groups);
    return check_hip(e) ? FL_ATTN_OK : FL_ATTN_ERR_HIP;
}

int fl_kv8_evict(const fl_attn_desc *desc, const fl_kv8_cache *from, const fl_kv8_cache *to, const fl_kv8_evict_args *args_in, void *hip_stream)
{
    fl_attn_desc desc_copy;
    int st = import_desc(&desc, &desc_copy);
    if (st != FL_ATTN_OK) return st;
    fl_kv8_cache s, t;
    st = import_cache(desc, from, &s);
    if (st != FL_ATTN_OK) return st;
    fl_kv8_evict_args args;
    st = import_struct(args_in, &args, kEvictMinBytes);
    if (st != FL_ATTN_OK) return st;
    fl_attn_desc desc_to = *desc;
    if (args.to_total_len < 0 || args.reserved != 0) return FL_ATTN_ERR_ARGUMENT;
    if (args.to_total_len > 0) desc_to.total_len = args.to_total_len;
    st = validate_desc(&desc_to);
    if (st != FL_ATTN_OK) return st;
    st = import_cache(&desc_to, to, &t);
    if (st != FL_ATTN_OK) return st;
    if (!s.weights || !t.weights || !args.kept || !args.rows_out) return FL_ATTN_ERR_NULL_POINTER;
    for (const void *f : {(const void *)args.kept, (const void *)args.rows_out, (const void *)args.rows_per_seq})
        if ((reinterpret_cast<uintptr_t>(f) & 3u) != 0) return FL_ATTN_ERR_ALIGNMENT;
    // one workgroup writes rows_out while others still read rows_per_seq
    const size_t counts = (size_t)desc->batch_size * 4, listed = counts * desc->head_num * (size_t)(args.keep_blocks > 0 ? args.keep_blocks : 1);
    if (overlap(args.kept, listed, args.rows_out, counts) ||
        (args.rows_per_seq && (overlap(args.rows_per_seq, counts, args.rows_out, counts) || overlap(args.rows_per_seq, counts, args.kept, listed))))
        return FL_ATTN_ERR_ARGUMENT;
    if (s.block_len != t.block_len) return FL_ATTN_ERR_ARGUMENT;
    const int T = s.block_len, L = desc->total_len, L_to = desc_to.total_len, D = desc->size_per_head;
    if (!args.rows_per_seq && (args.rows < 0 || args.rows > L)) return FL_ATTN_ERR_POSITION;
    if (args.keep_blocks < 1 || args.keep_blocks > L_to / T || args.recent_blocks < 0 || args.recent_blocks > args.keep_blocks)
        return FL_ATTN_ERR_ARGUMENT;

    // `to` is the cache itself, or overlaps it nowhere
    const size_t bh = (size_t)desc->batch_size * desc->head_num;
    struct Range { const void *p; size_t n; };
    const size_t rows_from = bh * L * D, rows_to = bh * L_to * D, ent_from = bh * (L / T) * 4, ent_to = bh * (L_to / T) * 4, tail = bh * T * D * 2;
    const Range a[7] = {{s.k, rows_from}, {s.v, rows_from}, {s.k_scale, ent_from}, {s.v_scale, ent_from}, {s.weights, ent_from}, {s.k_tail, tail}, {s.v_tail, tail}};
    const Range b[7] = {{t.k, rows_to}, {t.v, rows_to}, {t.k_scale, ent_to}, {t.v_scale, ent_to}, {t.weights, ent_to}, {t.k_tail, tail}, {t.v_tail, tail}};
    int same = 0;
    for (int i = 0; i < 5; ++i) same += a[i].p == b[i].p;
    if (same != 0 && (same != 5 || L != L_to)) return FL_ATTN_ERR_ARGUMENT;
    const bool same_tails = s.k_tail == t.k_tail && s.v_tail == t.v_tail;
    for (int i = 0; i < 7; ++i)
        for (int j = 0; j < 7; ++j) {
            if (i == j && ((i < 5 && same == 5) || (i >= 5 && same_tails))) continue;
            if (overlap(a[i].p, a[i].n, b[j].p, b[j].n)) return FL_ATTN_ERR_ARGUMENT;
        }

    Kv8EvictParams p{};
    p.k8 = s.k; p.v8 = s.v; p.k_scale = s.k_scale; p.v_scale = s.v_scale; p.weights = s.weights;
    p.k_tail = static_cast<const _Float16 *>(s.k_tail); p.v_tail = static_cast<const _Float16 *>(s.v_tail);
    p.k8_to = t.k; p.v8_to = t.v; p.k_scale_to = t.k_scale; p.v_scale_to = t.v_scale; p.weights_to = t.weights;
    if (!same_tails) { p.k_tail_to = static_cast<_Float16 *>(t.k_tail); p.v_tail_to = static_cast<_Float16 *>(t.v_tail); }
    p.kept = args.kept; p.rows_to = args.rows_out; p.rows_per_seq = args.rows_per_seq; p.rows = args.rows;
    p.B = desc->batch_size; p.H = desc->head_num; p.D = D; p.T = T; p.t_shift = log2_of(T);
    p.nblk = L / T; p.nblk_to = L_to / T; p.keep = args.keep_blocks; p.recent = args.recent_blocks;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    // One launch, a workgroup per (b,h), where it has little to move or where there is one for every compute unit; else a
    // selection, then many workgroups for each.  Two launches / one, us: 15 (b,h) of 96 KB 6.5 / 6.5 and 3 less on the host, 8 of 16 KB
    // 5.8 / 5.0, 32 of 128 KB 6.8 / 7.4, of 256 KB 9.2 / 12.3, of 512 KB 13.8 / 24.5; 256 of 256 KB 29.4 / 27.6, 2048 208 / 195.
    if (args.keep_blocks <= flattn::kEvictListCap && ((int64_t)args.keep_blocks * T * D * 2 <= kEvictOneLaunchBytes || (int64_t)bh >= device_cus())) {
        if (!check_hip(launch(flattn::kv8_evict_kernel, dim3((unsigned)bh), dim3(flattn::kEvictThreads), stream, p))) return FL_ATTN_ERR_HIP;
        return FL_ATTN_OK;
    }
    const int slices = (T * D / 16 + 255) / 256;
    if ((int64_t)bh * 2 * slices > INT32_MAX / 128) return FL_ATTN_ERR_SHAPE;
    if (!check_hip(launch(flattn::kv8_select_kernel, dim3((unsigned)bh), dim3(256), stream, p))) return FL_ATTN_ERR_HIP;
    if (!check_hip(launch(flattn::kv8_move_kernel, dim3((unsigned)(bh * 2 * slices)), dim3(256), stream, p, slices))) return FL_ATTN_ERR_HIP;
    return FL_ATTN_OK;
}

} // extern "C"
