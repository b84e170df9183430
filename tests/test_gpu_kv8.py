"""The 8-bit key/value cache on the GPU, through the C ABI, against float64 (tests/kv8_reference.py).  Rows, scales and tails
are compared bit for bit, whole arrays, so that a store outside its place shows; what has not been written yet holds NaN."""
import math

import numpy as np
import pytest

from fasterllama_amd import capi, synth
import kv8_reference as kr

pytestmark = pytest.mark.gpu

NEG = -3.4028234663852886e38


def to_gpu(c, dev):
    import torch
    from fasterllama_amd.kv8 import KV8Cache
    return KV8Cache.of(c.T, *(torch.from_numpy(getattr(c, n).copy()).to(dev) for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")),
                       weights=None if c.weights is None else torch.from_numpy(c.weights.copy()).to(dev))


def bits(x):
    return np.ascontiguousarray(x).view({1: np.uint8, 2: np.uint16, 4: np.uint32}[x.dtype.itemsize])


def assert_cache(g, c, steps=1, rows=None):
    """rows: of the cache after a prompt.  A prompt that completes a block need not take its rows through the tail, as single
    steps do: behind the open block's rows a tail holds nothing."""
    for n in c.names():
        x, want = getattr(g, n).cpu().numpy(), getattr(c, n)
        if rows is not None and n.endswith("_tail"):
            x, want = x[:, :, :rows % c.T], want[:, :, :rows % c.T]
        if n == "weights":
            # a weight's relative error is that of the softmax (a few hundred U at the sizes here), per step
            ok = ~np.isnan(want)
            assert np.array_equal(np.isnan(x), ~ok), "weights: NaN elsewhere"
            assert (np.abs(x[ok] - want[ok]) <= 2e-5 * steps * np.maximum(1.0, np.abs(want[ok]))).all(), np.abs(x[ok] - want[ok]).max()
        else:
            bad = np.flatnonzero(bits(x).ravel() != bits(want).ravel())
            assert bad.size == 0, f"{n}: {bad.size} of {x.size} differ, first at {np.unravel_index(bad[0], x.shape)}"


def assert_out(got, want, tol, what=""):
    got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    err = np.where(np.isnan(want), 0.0, np.abs(got - want))
    print(f"{what}: max error {err.max():.2e}, of the tolerance {np.max(err / np.maximum(tol, 1e-300)):.3f}")
    assert (err <= tol).all(), f"{what}: {err.max()} against {np.max(tol)}"


def inputs(B, S, H, D, dtype, seed):
    r = np.random.RandomState(seed)
    if dtype == "i32":
        acc = [r.randint(-40000, 40000, (B, S, H, D)).astype(np.int32) for _ in range(3)]
        sc = [(r.rand(B, S) * 2e-3 + 1e-4).astype(np.float32)] + [(r.rand(H * D) * 0.05 + 0.01).astype(np.float32) for _ in range(3)]
        val = [((a.astype(np.float32) * sc[0][..., None, None]) * w.reshape(H, D)).astype(np.float32) for a, w in zip(acc, sc[1:])]
        return acc, val, sc
    x = [r.randn(B, S, H, D).astype(np.float16 if dtype == "f16" else np.float32) for _ in range(3)]
    return x, x, None


def masks(kind, L, seed=0):
    i = np.arange(L)
    if kind is None:
        return None
    if kind == "causal":
        return np.where(i[None] > i[:, None], np.float32(NEG), np.float32(0)).astype(np.float32)
    if kind == "inf_window":  # -inf outside the last 40 columns
        return np.where((i[None] > i[:, None]) | (i[None] + 40 < i[:, None]), np.float32(-np.inf), np.float32(0)).astype(np.float32)
    if kind == "soft":
        return np.where(i[None] > i[:, None], np.float32(-1e5), np.random.RandomState(seed).randn(L, L)).astype(np.float32)
    if kind == "strict":  # the first row sees nothing
        return np.where(i[None] >= i[:, None], np.float32(NEG), np.float32(0)).astype(np.float32)
    raise KeyError(kind)


class Case:
    def __init__(self, dev, B, H, D, L, T, dtype="f16", rows=0, weights=False, nsplit=0, max_seq_len=1, seed=0, scale=0.0):
        import torch
        from fasterllama_amd.kv8 import KV8Attention
        self.dev, self.B, self.H, self.D, self.L, self.T, self.dtype, self.seed = dev, B, H, D, L, T, dtype, seed
        self.scale = scale
        self.rows = np.full(B, rows) if np.isscalar(rows) else np.asarray(rows)
        self.ref = kr.Cache(B, H, D, L, T, weights, seed=seed).fill(np.clip(self.rows, 0, L - 1), seed + 1)
        self.gpu = to_gpu(self.ref, dev)
        self.table = synth.freq_cis_table(L + 64, D)
        self.table_d = torch.from_numpy(self.table).to(dev)
        self.op = KV8Attention(B, H, D, L, torch.float16 if dtype == "f16" else torch.float32, T, max_seq_len, nsplit, scale, dev)

    def t(self, x):
        import torch
        return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(self.dev)

    def feed(self, S, seed):
        raw, val, sc = inputs(self.B, S, self.H, self.D, self.dtype, seed)
        return [self.t(x) for x in raw], val, None if sc is None else tuple(self.t(x) for x in sc)

    def decode(self, mask=None, ragged=False, rope=None, seed=7, bound=None, **kw):
        raw, val, sc = self.feed(1, seed)
        if ragged:
            kw.update(start_pos_per_seq=self.t(self.rows.astype(np.int32)), max_start_pos=int(self.rows.max()) if bound is None else bound)
        else:
            kw.update(start_pos=int(self.rows[0]))
        if rope is not None:
            kw.update(rope_row_per_seq=self.t(np.asarray(rope, np.int32)))
        got = self.op.decode(*raw, self.gpu, self.table_d, attn_mask=self.t(mask), scales=sc, **kw)
        start = self.rows if bound is None else np.where(self.rows > bound, -1, self.rows)
        want, tol = self.ref.step(*val, self.table, start, mask, rope, self.scale)
        return got, want[:, :, 0], tol[..., 0]

    def prompt(self, S, mask=None, seed=9, weight_queries=0, **kw):
        raw, val, sc = self.feed(S, seed)
        got = self.op.prefill(*raw, self.gpu, self.table_d, start_pos=int(self.rows[0]), attn_mask=self.t(mask), scales=sc,
                              weight_queries=weight_queries, **kw)
        want, tol = self.ref.step(*val, self.table, self.rows, mask, None, self.scale, weight_queries)
        return got, want, tol


# ------------------------------------------------------------------------------------------------------------- decode

@pytest.mark.parametrize("D", [32, 64, 96, 128, 256, 512, 1024])
@pytest.mark.parametrize("T", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_decode_head_sizes(gpu, D, T, dtype):
    for rows in (0, 1, T - 1, T, 2 * T + 5, 3 * T - 1):
        c = Case(gpu, 2, 3, D, 3 * T if T == 128 else 4 * T, T, dtype, rows, weights=True)
        got, want, tol = c.decode()
        assert_out(got, want, tol, f"rows {rows}")
        assert_cache(c.gpu, c.ref)


@pytest.mark.parametrize("kind", ["causal", "inf_window", "soft"])
@pytest.mark.parametrize("rows", [31, 63, 200, 383])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_decode_masks(gpu, kind, rows, nsplit):
    c = Case(gpu, 2, 2, 64, 512, 32, "f32", rows, weights=True, nsplit=nsplit)
    got, want, tol = c.decode(masks(kind, 512))
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref)


@pytest.mark.parametrize("D,rows", [(128, 0), (96, 70)])
def test_a_row_that_sees_nothing_is_nan_and_gathers_nothing(gpu, D, rows):
    m = np.full((128, 128), NEG, np.float32)
    for value in (NEG, -np.inf):
        m[:] = value
        c = Case(gpu, 1, 2, D, 128, 64, "f16", rows, weights=True)
        before = c.ref.weights.copy()
        got, want, tol = c.decode(m)
        assert np.isnan(got.cpu().numpy()).all() and np.isnan(want).all()
        after = c.gpu.weights.cpu().numpy()
        n = rows // 64 + (rows % 64 > 0)
        assert np.array_equal(after[:, :, :n], before[:, :, :n])


@pytest.mark.parametrize("ready,nsplit", [(True, 1), (True, 3), (False, 3)])
@pytest.mark.parametrize("rows", [0, 64, 384])
def test_a_block_whose_first_row_sees_nothing_starts_from_zero(gpu, rows, ready, nsplit):
    c = Case(gpu, 2, 2, 64, 512, 64, "f16", rows, weights=True, nsplit=nsplit)  # (behind the rows the weights are NaN)
    if not ready:  # the merge as a launch of its own
        def without(call, *args):
            c.op.io.flags = 0
            capi.check(call(*args, 0))
        c.op._enqueue = without
    got, want, tol = c.decode(np.full((512, 512), NEG, np.float32))
    assert np.isnan(got.cpu().numpy()).all()
    assert_cache(c.gpu, c.ref)
    assert not c.gpu.weights[:, :, rows // 64].cpu().numpy().any()


@pytest.mark.parametrize("ready", [True, False])
@pytest.mark.parametrize("nsplit", [0, 2, 7, 1024])
def test_decode_splits(gpu, nsplit, ready):
    c = Case(gpu, 1, 2, 128, 2048, 64, "f16", 2000, weights=True, nsplit=nsplit)
    if not ready:  # two launches
        def without(call, *args):
            c.op.io.flags = 0
            capi.check(call(*args, 0))
        c.op._enqueue = without
    import torch
    torch.cuda.synchronize()
    for step in range(2):  # the counters are zero again for the second
        c.rows[:] = 2000 + step
        got, want, tol = c.decode(seed=step)
        torch.cuda.synchronize()
        assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref, 2)


def test_decode_from_an_empty_cache_over_block_borders(gpu):
    c = Case(gpu, 2, 2, 96, 96, 32, "f16", 0, weights=True)
    for step in range(96):
        c.rows[:] = step
        got, want, tol = c.decode(seed=100 + step)
        assert_out(got, want, tol, f"step {step}")
    assert_cache(c.gpu, c.ref, 96)


@pytest.mark.parametrize("dtype", ["f16", "i32"])
@pytest.mark.parametrize("nsplit", [0, 4])
def test_decode_ragged_with_positions_outside(gpu, dtype, nsplit):
    rows = np.array([0, 511, 31, 600, -1, 63, 64, 200, 640, 450])
    c = Case(gpu, 10, 3, 64, 640, 32, dtype, rows, weights=True, nsplit=nsplit)
    got, want, tol = c.decode(ragged=True, bound=599, rope=np.array([5, 0, 1, 2, 3, 4, 5, 100, 7, 650]))
    assert_out(got, want, tol)
    assert np.isnan(got.cpu().numpy()[[3, 4, 8]]).all()
    assert_cache(c.gpu, c.ref)


def test_table_rows_outside_the_table_store_nothing(gpu):
    for nsplit in (1, 3):
        c = Case(gpu, 4, 2, 64, 640, 32, "f16", [500, 501, 502, 503], weights=True, nsplit=nsplit)
        before = c.ref.copy()
        raw, val, _ = c.feed(1, 7)
        rope = np.array([704, 703, -1, 2 ** 31 - 1])  # the table has 704 rows
        got = c.op.decode(*raw, c.gpu, c.table_d, start_pos_per_seq=c.t(c.rows.astype(np.int32)), max_start_pos=503, rope_row_per_seq=c.t(rope.astype(np.int32)))
        want, tol = c.ref.step(*val, c.table, [-1, 501, -1, -1], rope=rope)
        assert_out(got, want[:, :, 0], tol[..., 0])
        assert_cache(c.gpu, c.ref)


def test_two_objects_on_two_streams(gpu):
    """Each has its workspace: split steps side by side."""
    import torch
    cases = [Case(gpu, 1, 8, 128, 4096, 64, "f16", 4000 + 63 * i, weights=True, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream(gpu) for _ in cases]
    torch.cuda.synchronize()
    feeds = [c.feed(1, 5) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, (raw, _, _) in zip(cases, streams, feeds):
            with torch.cuda.stream(s):
                c.gpu.weights.zero_()
                c.got = c.op.decode(*raw, c.gpu, c.table_d, start_pos=int(c.rows[0]))
    torch.cuda.synchronize()
    for c, (_, val, _) in zip(cases, feeds):
        c.ref.weights[:] = 0
        want, tol = c.ref.step(*val, c.table, c.rows)
        assert_out(c.got, want[:, :, 0], tol[..., 0])
        assert_cache(c.gpu, c.ref)


def test_wrapper_refusals(gpu):
    import torch
    c = Case(gpu, 2, 2, 64, 128, 32, "f16", 5, weights=True, max_seq_len=16)
    (q, k, v), _, _ = c.feed(1, 1)
    bad = [dict(q=q.float()), dict(q=q[:, :, :1]), dict(q=q.transpose(2, 3)), dict(q=q.cpu()), dict(freq=c.table_d[:4]), dict(freq=c.table_d[:, :32]),
           dict(attn_mask=torch.zeros(3, 128, device=gpu)), dict(attn_mask=torch.zeros(128, 5, device=gpu)), dict(attn_mask=torch.zeros(128, 128, device=gpu).t()),
           dict(start_pos=128), dict(start_pos=-1), dict(start_pos_per_seq=torch.zeros(3, dtype=torch.int32, device=gpu)),
           dict(start_pos_per_seq=torch.zeros(2, dtype=torch.int64, device=gpu)), dict(out=torch.empty(2, 64, device=gpu)),
           dict(cache=to_gpu(kr.Cache(2, 2, 64, 160, 32), gpu)), dict(cache=to_gpu(kr.Cache(2, 2, 64, 128, 64), gpu))]
    for kw in bad:
        a = {"q": q, "cache": c.gpu, "freq": c.table_d, "start_pos": 5, **kw}
        rest = {n: x for n, x in a.items() if n not in ("q", "cache", "freq")}
        with pytest.raises(capi.FlAttnError):
            c.op.decode(a["q"], k, v, a["cache"], a["freq"], **rest)
    (q, k, v), _, _ = c.feed(17, 1)
    with pytest.raises(capi.FlAttnError):
        c.op.prefill(q, k, v, c.gpu, c.table_d)
    (q, k, v), _, _ = c.feed(16, 1)
    with pytest.raises(capi.FlAttnError):
        c.op.prefill(q, k, v, c.gpu, c.table_d, start_pos=113)
    with pytest.raises(capi.FlAttnError):
        c.op.prefill(q, k, v, c.gpu, c.table_d, mask_tile_classes=torch.zeros(7, dtype=torch.uint8, device=gpu))
    for rows in (0, 129):
        with pytest.raises(capi.FlAttnError):
            c.op.read(c.gpu, rows)
    for keep, recent, rows in ((0, 0, 64), (5, 0, 64), (2, 3, 64), (2, 1, 129)):
        with pytest.raises(capi.FlAttnError):
            c.op.evict(c.gpu, keep, recent, rows)
    with pytest.raises(capi.FlAttnError):
        c.op.evict(to_gpu(kr.Cache(2, 2, 64, 128, 32), gpu), 1, 0, 64)
    torch.cuda.synchronize()


def test_decode_scales_of_stale_blocks_and_rows_are_never_read(gpu):
    """The whole cache behind the rows is NaN scales and random integers (Cache's junk): the last trip of a wave reaches over
    the last complete block at head sizes whose trips are longer than a block."""
    for D in (32, 64):
        c = Case(gpu, 1, 1, D, 512, 32, "f16", 33, weights=True)
        got, want, tol = c.decode()
        assert_out(got, want, tol)


def test_non_finite_inputs_do_not_spread(gpu):
    """A NaN or infinity in a key or value is stored as 0; in a query it makes that head's output NaN."""
    import torch
    for rows in (10, 31):
        c = Case(gpu, 1, 3, 64, 64, 32, "f32", rows)
        raw, val, _ = c.feed(1, 3)
        q, k, v = (x.copy() for x in val)
        k[0, 0, 0, 5], k[0, 0, 1, 6], v[0, 0, 0, 7], v[0, 0, 2, 8] = np.nan, np.inf, -np.inf, 1e30
        q[0, 0, 1, 3] = np.nan
        got = c.op.decode(c.t(q), c.t(k), c.t(v), c.gpu, c.table_d, start_pos=rows)
        want, tol = c.ref.step(q, k, v, c.table, c.rows)
        assert np.isnan(got.cpu().numpy().reshape(3, 64)[1]).all()
        assert_out(got.view(1, 3, 64)[:, [0]], want[:, [0], 0], tol[..., 0])
        assert_cache(c.gpu, c.ref)


def test_decode_int8_output_and_int32_input(gpu):
    import torch
    c = Case(gpu, 3, 4, 128, 256, 64, "i32", 190)
    q8, sc = torch.zeros(3, 512, dtype=torch.int8, device=gpu), torch.zeros(3, device=gpu)
    out = torch.empty(3, 512, device=gpu)
    _, want, tol = c.decode(out=out, out_int8=q8, out_scale=sc)
    assert_out(out, want, tol)
    x = out.cpu().numpy()
    top = np.abs(x).max(1)
    assert np.array_equal(sc.cpu().numpy(), top / np.float32(127))
    assert np.array_equal(q8.cpu().numpy(), np.rint((x * np.float32(127)) / top[:, None]).astype(np.int8))


# ------------------------------------------------------------------------------------------------------------- prompt

@pytest.mark.parametrize("D", [32, 64, 96, 128, 256, 512, 1024])
@pytest.mark.parametrize("T,dtype", [(32, "f32"), (64, "f16"), (128, "f16")])
def test_prompt_head_sizes(gpu, D, T, dtype):
    for start, S in ((0, 1), (0, T), (5, 2 * T), (T, 17), (T - 1, T + 2)):
        c = Case(gpu, 2, 2, D, 4 * T, T, dtype, start, weights=D <= 128, max_seq_len=S)
        got, want, tol = c.prompt(S, masks("causal", 4 * T))
        assert_out(got, want, tol, f"start {start} S {S}")
        assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("kind", [None, "causal", "inf_window", "soft", "strict"])
@pytest.mark.parametrize("start,S", [(0, 300), (77, 333), (64, 128), (130, 1)])
def test_prompt_masks(gpu, kind, start, S):
    c = Case(gpu, 1, 3, 128, 448, 64, "f16", start, weights=True, max_seq_len=S)
    got, want, tol = c.prompt(S, masks(kind, 448), weight_queries=50)
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("D,T,dtype", [(128, 64, "f16"), (96, 32, "f32"), (32, 128, "i32"), (256, 64, "f16")])
@pytest.mark.parametrize("kind", [None, "causal"])
@pytest.mark.parametrize("start,S", [(0, 300), (77, 130), (13, 60), (1100, 40)])
def test_padded_prompts_of_different_lengths(gpu, D, T, dtype, kind, start, S):
    """The padding (NaN here) is neither stored nor read; rows behind a sequence's own are left as they were."""
    import torch
    lens = np.array([S, 0, 1, S // 2, S + 1, -1, 32, S - 1], np.int32)
    L = 1152 if start > 1000 else 384
    c = Case(gpu, 8, 2, D, L, T, dtype, start, weights=D <= 128, max_seq_len=S)
    raw, val, sc = c.feed(S, 11)
    for b in range(8):
        for x in raw:
            x[b, max(lens[b], 0):] = 2 ** 30 if dtype == "i32" else float("nan")
    m = masks(kind, L)
    before = {n: getattr(c.gpu, n).cpu().numpy().copy() for n in c.ref.names()}
    got = c.op.prefill(*raw, c.gpu, c.table_d, start_pos=start, attn_mask=c.t(m), scales=sc, weight_queries=20, seq_len_per_seq=c.t(lens))
    want, tol = c.ref.step(*val, c.table, c.rows, m, weight_queries=20, lens=lens)
    assert_out(got, want, tol, f"D {D} start {start} S {S}")
    for b in range(8):
        assert not got[b, :, max(lens[b], 0):].cpu().numpy().any() or lens[b] not in range(S + 1)
    n = np.where((lens < 0) | (lens > S), 0, lens) + start
    for b in range(8):
        for name in c.ref.names():
            x, ref = getattr(c.gpu, name)[b].cpu().numpy(), getattr(c.ref, name)[b]
            if name == "weights":
                ok = ~np.isnan(ref)
                assert np.array_equal(np.isnan(x), ~ok) and (np.abs(x[ok] - ref[ok]) <= 2e-5 * 20 * np.maximum(1.0, np.abs(ref[ok]))).all(), b
            elif name.endswith("_tail"):
                assert np.array_equal(bits(x[:, :n[b] % T]), bits(ref[:, :n[b] % T])), (b, name)
            else:
                assert np.array_equal(bits(x), bits(ref)), (b, name)
    # and every sequence decodes on from its own length
    c.rows = np.where((lens < 0) | (lens > S), -1, n)
    got, want, tol = c.decode(ragged=True, seed=12, bound=start + S)
    assert_out(got, want, tol, "step")


@pytest.mark.parametrize("dtype", ["f16", "i32"])
def test_prompt_in_pieces_and_steps_leaves_the_same_bits(gpu, dtype):
    """Rows, scales and tails do not depend on how the rows arrived."""
    S, pieces = 150, (40, 24, 1, 64, 21)
    for T in (32, 128):
        one = Case(gpu, 2, 2, 64, 256, T, dtype, 0, max_seq_len=S)
        raw, val, sc = one.feed(S, 5)
        one.op.prefill(*raw, one.gpu, one.table_d, scales=sc)
        two = Case(gpu, 2, 2, 64, 256, T, dtype, 0, max_seq_len=S)
        at = 0
        for n in pieces:
            part = [x[:, at:at + n].contiguous() for x in raw]
            psc = None if sc is None else (sc[0][:, at:at + n].contiguous(), *sc[1:])
            if n == 1:
                two.op.decode(*part, two.gpu, two.table_d, start_pos=at, scales=psc)
            else:
                two.op.prefill(*part, two.gpu, two.table_d, start_pos=at, scales=psc)
            at += n
        one.ref.step(*val, one.table, [0, 0])
        for c in (one, two):
            for n in ("k", "v", "k_scale", "v_scale"):
                m = 150 // T * (T if n in ("k", "v") else 1)
                assert np.array_equal(bits(getattr(c.gpu, n).cpu().numpy()[:, :, :m]), bits(getattr(one.ref, n)[:, :, :m])), n
            for n in ("k_tail", "v_tail"):
                assert np.array_equal(bits(getattr(c.gpu, n).cpu().numpy()[:, :, :150 % T]), bits(getattr(one.ref, n)[:, :, :150 % T])), n


def test_prompt_scores_of_every_size(gpu):
    """Keys and queries of very different sizes, block to block: the scales and the running maximum have to keep up."""
    c = Case(gpu, 1, 2, 128, 512, 32, "f32", 0, max_seq_len=400, weights=True)
    raw, val, _ = c.feed(400, 3)
    r = np.random.RandomState(0)
    q, k, v = (x.copy() for x in val)
    k *= np.exp2(r.randint(-6, 4, (1, 400, 1, 1))).astype(np.float32)
    v *= np.exp2(r.randint(-12, 8, (1, 400 // 16, 1, 1)).repeat(16, 1)).astype(np.float32)
    q *= np.exp2(r.randint(-4, 3, (1, 400, 1, 1))).astype(np.float32)
    m = masks("causal", 512)
    got = c.op.prefill(c.t(q), c.t(k), c.t(v), c.gpu, c.table_d, attn_mask=c.t(m))
    want, tol = c.ref.step(q, k, v, c.table, c.rows, m)
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref, 400, 400)


@pytest.mark.parametrize("D,T,dtype", [(128, 64, "f16"), (96, 32, "f32"), (32, 128, "f16")])
@pytest.mark.parametrize("kind", [None, "causal", "inf_window", "strict"])
def test_prompt_pieces_behind_a_long_context_share_their_keys(gpu, D, T, dtype, kind):
    """Few queries, many keys: the keys are split over workgroups, some of which a window leaves nothing."""
    for start, S in ((1301, 3), (1100, 130), (0, 1)):
        c = Case(gpu, 1, 2, D, 1536, T, dtype, start, weights=True, max_seq_len=200)
        got, want, tol = c.prompt(S, masks(kind, 1536), weight_queries=2)
        assert_out(got, want, tol, f"start {start} S {S}")
        assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("kind", [None, "padding"])
def test_prompt_over_more_tiles_than_one_list(gpu, kind):
    """33 100 keys: the tile list is built twice."""
    import torch
    c = Case(gpu, 1, 1, 32, 128 * 259, 128, "f16", 0, max_seq_len=64, weights=True)
    r = np.random.RandomState(0)
    n, start, S = 128 * 259, 33060, 40
    c.ref.k_scale[:], c.ref.v_scale[:], c.ref.weights[:] = 0.01 + 0.02 * r.rand(1, 1, 259), 0.01 + 0.02 * r.rand(1, 1, 259), 0
    c.ref.k_tail[:], c.ref.v_tail[:] = r.randn(1, 1, 128, 32), r.randn(1, 1, 128, 32)
    c.gpu, c.rows = to_gpu(c.ref, gpu), np.array([start])
    raw, val, _ = c.feed(S, 5)
    m = None
    if kind:
        m = np.zeros((1, n), np.float32)
        m[0, :1000], m[0, 20000:30000] = NEG, -np.inf
    got = c.op.prefill(*raw, c.gpu, c.table_d, start_pos=start, attn_mask=c.t(m), weight_queries=7)
    want, tol = c.ref.step(*val, c.table, [start], None if m is None else np.broadcast_to(m, (n, n)), weight_queries=7)
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("H", [1, 8])
def test_block_weights_of_more_queries_than_one_list(gpu, H):
    """33 000 queries: the list of query blocks is built twice (8 heads: with the operands staged)."""
    import torch
    from fasterllama_amd.decode_attn import rope_table
    from fasterllama_amd.kv8 import KV8Attention, KV8Cache
    S, L, D, T, W = 33000, 33024, 32, 128, 32990
    g = torch.Generator(device=gpu).manual_seed(0)
    q, k, v = (torch.randn(1, S, H, D, generator=g, device=gpu, dtype=torch.float32) for _ in range(3))
    table, cache = rope_table(L, D, device=gpu), KV8Cache(1, H, D, L, T, weights=True, device=gpu)
    op = KV8Attention(1, H, D, L, torch.float32, T, max_seq_len=S, device=gpu)
    op.prefill(q, k, v, cache, table, weight_queries=W)
    keys, _ = op.read(cache, S)
    x, f = q[0].double(), table[:S, None].double()
    rot = torch.stack([x[..., 0::2] * f[..., 0::2] - x[..., 1::2] * f[..., 1::2], x[..., 1::2] * f[..., 0::2] + x[..., 0::2] * f[..., 1::2]], -1).flatten(-2)
    for h in range(H):
        want = torch.zeros(L // T * T, dtype=torch.float64, device=gpu)
        for q0 in range(S - W, S, 2000):
            z = rot[q0:q0 + 2000, h] @ keys[0, h].double().T / math.sqrt(D)
            want[:S] += torch.softmax(z, -1).sum(0)
        want = want.view(-1, T).sum(-1)
        # every weight is off by its softmax's relative error, a few hundred units of 2^-24 as in assert_cache
        assert ((cache.weights[0, h].double() - want).abs() <= 2e-5 * want).all()


def test_graph_of_a_prompt_an_eviction_and_a_read(gpu):
    """Captured once, replayed with eager work between: every replay equals the eager run."""
    import torch
    c = Case(gpu, 2, 4, 128, 512, 64, "f16", 70, weights=True, max_seq_len=300)
    m = c.t(masks("causal", 512))
    raw, _, _ = c.feed(300, 3)
    start = to_gpu(c.ref, gpu)
    names = c.ref.names()

    def restore():
        for n in names:
            getattr(c.gpu, n).copy_(getattr(start, n))

    def run():
        out = c.op.prefill(*raw, c.gpu, c.table_d, start_pos=70, attn_mask=m, weight_queries=100)
        kept, rows = c.op.evict(c.gpu, 3, 1, 370)
        return (out, kept, rows, *c.op.read(c.gpu, 3 * 64 + 370 % 64))
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        want = [x.clone() for x in run()]
        state = {n: getattr(c.gpu, n).clone() for n in names}
    torch.cuda.synchronize()
    restore()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for _ in range(4):
        restore()
        for x in got:
            x.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        for n in names:
            assert torch.equal(getattr(c.gpu, n).float().nan_to_num(7.0), state[n].float().nan_to_num(7.0)), n


def test_non_finite_prompt_inputs_do_not_spread(gpu):
    c = Case(gpu, 1, 2, 64, 256, 32, "f32", 0, max_seq_len=100)
    raw, val, _ = c.feed(100, 3)
    q, k, v = (x.copy() for x in val)
    k[0, 3, 0, 5], k[0, 40, 1, 6], v[0, 99, 0, 7], v[0, 70, 1, 8], v[0, 2, 1, 0] = np.nan, np.inf, -np.inf, 1e30, np.nan
    q[0, 50, 1, 3], q[0, 51, 0, 0] = np.nan, np.inf
    m = masks("causal", 256)
    got = c.op.prefill(c.t(q), c.t(k), c.t(v), c.gpu, c.table_d, attn_mask=c.t(m))
    with np.errstate(invalid="ignore"):
        want, tol = c.ref.step(q, k, v, c.table, c.rows, m)
    assert np.isnan(want[0, 1, 50]).all() and np.isnan(want[0, 0, 51]).all()
    assert_out(got[:, [0]], want[:, [0]], tol)  # (head 1's 65504 is a scale of its own)
    assert_cache(c.gpu, c.ref, 100, 100)


def test_prompt_with_a_persistent_class_table_and_int8_output(gpu):
    import torch
    from fasterllama_amd.decode_attn import PrefillAttention
    c = Case(gpu, 2, 3, 128, 512, 64, "f16", 96, max_seq_len=300)
    m = masks("causal", 512)
    md = c.t(m)
    table = PrefillAttention(2, 3, 128, 512, 300, torch.float16, device=gpu).classify_mask(md)
    q8, sc = torch.zeros(2, 300, 384, dtype=torch.int8, device=gpu), torch.zeros(2, 300, device=gpu)
    out = torch.empty(2, 3, 300, 128, device=gpu)
    _, want, tol = c.prompt(300, m, mask_tile_classes=table, out=out, out_int8=q8, out_scale=sc)
    assert_out(out, want, tol)
    x = out.cpu().numpy().transpose(0, 2, 1, 3).reshape(2, 300, 384)
    top = np.abs(x).max(-1)
    assert np.array_equal(sc.cpu().numpy(), top / np.float32(127))
    assert np.array_equal(q8.cpu().numpy(), np.rint((x * np.float32(127)) / top[..., None]).astype(np.int8))


# --------------------------------------------------------------------------------------------------------- read, evict

@pytest.mark.parametrize("D,T,dtype", [(32, 32, "f32"), (96, 64, "f16"), (128, 128, "f32"), (1024, 32, "f16")])
def test_read(gpu, D, T, dtype):
    rows = np.array([0, 1, T, T + 3, 2 * T + T // 2, 3 * T])
    c = Case(gpu, 6, 2, D, 3 * T, T, dtype, np.minimum(rows, 3 * T - 1))
    rows = c.rows
    for n in (1, T + 1, 3 * T):
        for ragged in (True, False):
            lens = np.minimum(rows if ragged else np.full(6, n), n)
            if not ragged and n > rows.min():
                continue
            k, v = c.op.read(c.gpu, n, c.t(rows.astype(np.int32)) if ragged else None)
            for b in range(6):
                # (a row of a block that the sequence has completed is a byte row, wherever the output ends)
                for x, want in zip((k, v), c.ref.values(b, int(rows[b]))):
                    x = x[b].cpu().numpy()
                    assert not x[:, lens[b]:].any()
                    want = want[:, :lens[b]].astype(np.float32).astype(x.dtype)
                    # (the fp16 value is that of the 32-bit product)
                    assert np.array_equal(x[:, :lens[b]], want)


@pytest.mark.parametrize("D,T", [(32, 32), (96, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (3, 3), (5, 2), (7, 1), (9, 4)])
def test_evict(gpu, D, T, keep, recent):
    L = 9 * T
    rows = np.array([0, 3 * T, 7 * T + 5, 9 * T - 1, T - 1, -1, 9 * T + 1])
    for place in ("in place", "same size", "smaller"):
        c = Case(gpu, 7, 2, D, L, T, "f16", rows, weights=True)
        r = np.random.RandomState(keep)
        w = c.ref.weights
        w[:] = r.randint(0, 4, w.shape)  # ties
        w[0, 0, 1], w[2, 1, 3], w[3, 0, :] = np.nan, np.nan, np.inf
        w[3, 1, :] = -0.0
        w[3, 1, 2::3] = 0.0
        c.gpu = to_gpu(c.ref, gpu)
        into = None if place == "in place" else kr.Cache(7, 2, D, L if place == "same size" else keep * T, T, True, seed=5)
        to = None if into is None else to_gpu(into, gpu)
        kept, after = c.op.evict(c.gpu, keep, recent, 0, c.t(rows.astype(np.int32)), into=to)
        want_kept, want_after = kr.evict(c.ref, rows, keep, recent, into)
        assert np.array_equal(kept.cpu().numpy(), want_kept), (kept.cpu().numpy() != want_kept).any(-1)
        assert np.array_equal(after.cpu().numpy(), want_after)
        g, want = (c.gpu, c.ref) if into is None else (to, into)
        for n in want.names():
            assert np.array_equal(bits(getattr(g, n).cpu().numpy()), bits(getattr(want, n))), (place, n)


def test_read_of_fewer_rows_than_a_sequence_holds(gpu):
    c = Case(gpu, 3, 2, 64, 192, 64, "f32", np.array([100, 191, 20]))
    for n in (1, 40, 64, 70, 130):
        k, v = c.op.read(c.gpu, n, c.t(c.rows.astype(np.int32)))
        for b in range(3):
            for x, want in zip((k, v), c.ref.values(b, int(c.rows[b]))):
                m = min(n, int(c.rows[b]))
                x = x[b].cpu().numpy()
                assert np.array_equal(x[:, :m], want.astype(np.float32)[:, :m]) and not x[:, m:].any()


def test_evict_many_blocks(gpu):
    """More blocks than threads: weights over 30 binary orders, and all but equal ones."""
    for spread in (True, False):
        c = Case(gpu, 2, 2, 32, 32 * 1500, 32, "f16", 0, weights=True)
        r = np.random.RandomState(1)
        c.ref.weights[:] = np.exp2(r.uniform(-15, 15, c.ref.weights.shape)) if spread else 1.0 + r.randint(0, 3, c.ref.weights.shape) * 2.0 ** -23
        c.ref.k_scale[:], c.ref.v_scale[:] = r.rand(*c.ref.k_scale.shape), r.rand(*c.ref.k_scale.shape)
        c.gpu = to_gpu(c.ref, gpu)
        rows = np.full(2, 32 * 1500)
        kept, after = c.op.evict(c.gpu, 700, 100, 32 * 1500)
        want_kept, want_after = kr.evict(c.ref, rows, 700, 100)
        assert np.array_equal(kept.cpu().numpy(), want_kept)
        assert_cache(c.gpu, c.ref)


@pytest.mark.parametrize("B,H,D,T,blocks,keep,recent", [
    (2, 2, 32, 32, 1500, 60, 7),     # one launch, more blocks than its threads, chosen by histograms
    (16, 16, 128, 128, 7, 5, 1),     # a workgroup for every compute unit
    (3, 2, 64, 64, 66, 20, 2),       # 64 candidates, counted; two launches
    (3, 2, 64, 64, 67, 20, 2)])      # 65, by histograms
@pytest.mark.parametrize("place", ["in place", "other"])
def test_evict_by_either_way(gpu, B, H, D, T, blocks, keep, recent, place):
    c = Case(gpu, B, H, D, T * (blocks + 1), T, "f16", 0, weights=True)
    r = np.random.RandomState(blocks)
    c.ref.weights[:] = r.randint(0, 9, c.ref.weights.shape)
    c.ref.k_scale[:], c.ref.v_scale[:] = r.rand(*c.ref.k_scale.shape), r.rand(*c.ref.k_scale.shape)
    c.ref.k_tail[:], c.ref.v_tail[:] = r.rand(*c.ref.k_tail.shape), r.rand(*c.ref.k_tail.shape)
    into = None if place == "in place" else kr.Cache(B, H, D, T * (keep + 1), T, True, seed=5)
    c.gpu, to = to_gpu(c.ref, gpu), None if into is None else to_gpu(into, gpu)
    rows = T * blocks + 3
    kept, after = c.op.evict(c.gpu, keep, recent, rows, into=to)
    want_kept, want_after = kr.evict(c.ref, np.full(B, rows), keep, recent, into)
    assert np.array_equal(kept.cpu().numpy(), want_kept) and np.array_equal(after.cpu().numpy(), want_after)
    g, want = (c.gpu, c.ref) if into is None else (to, into)
    for n in want.names():
        assert np.array_equal(bits(getattr(g, n).cpu().numpy()), bits(getattr(want, n))), n


@pytest.mark.parametrize("T", [32, 64])
def test_serving_run(gpu, T):
    """Prompt, steps, eviction in place, steps: as a server would, with the budget of a small cache."""
    L = 8 * T
    c = Case(gpu, 2, 3, 64, L, T, "f16", 0, weights=True, max_seq_len=7 * T)
    m = masks("causal", L)
    got, want, tol = c.prompt(6 * T + 7, m, weight_queries=33)
    assert_out(got, want, tol, "prompt")
    rows, pos, steps = 6 * T + 7, 6 * T + 7, 33
    for step in range(4 * T):
        if rows == L:
            # the weights decide as they stand here: those of the GPU and of the reference differ in their last bits
            c.ref.weights[:] = c.gpu.weights.cpu().numpy()
            kept, after = c.op.evict(c.gpu, 5, 2, rows)
            want_kept, _ = kr.evict(c.ref, np.full(2, rows), 5, 2)
            assert np.array_equal(kept.cpu().numpy(), want_kept)
            rows = 5 * T
            assert (after.cpu().numpy() == rows).all()
        c.rows[:] = rows
        got, want, tol = c.decode(seed=1000 + step, rope=[pos, pos]) if step % 2 else c.decode(seed=1000 + step, rope=[pos, pos], ragged=True)
        assert_out(got, want, tol, f"step {step} row {rows}")
        rows, pos, steps = rows + 1, min(pos + 1, L + 63), steps + 1
    assert_cache(c.gpu, c.ref, steps)


# ---------------------------------------------------------------------------------------------- streams, graphs, limits

def test_side_stream_and_graph_replays(gpu):
    """A captured step, replayed with eager work between: every replay equals the eager result."""
    import torch
    c = Case(gpu, 1, 4, 128, 2048, 64, "f16", 1983, weights=True)  # a split context, a block filled
    m = c.t(masks("causal", 2048))
    raw, _, _ = c.feed(1, 3)
    start = to_gpu(c.ref, gpu)
    names = c.ref.names()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        want = c.op.decode(*raw, c.gpu, c.table_d, start_pos=1983, attn_mask=m).clone()
        want_state = {n: getattr(c.gpu, n).clone() for n in names}
    side.synchronize()

    def restore():
        for n in names:
            getattr(c.gpu, n).copy_(getattr(start, n))
    restore()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.op.decode(*raw, c.gpu, c.table_d, start_pos=1983, attn_mask=m)
    for _ in range(4):
        restore()
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for n in names:
            assert torch.equal(getattr(c.gpu, n).float().nan_to_num(7.0), want_state[n].float().nan_to_num(7.0)), n


def test_caches_past_four_gib(gpu):
    """Offsets of whole caches pass 32 bits: 2 x 4.3 GB of bytes, the last sequence's last rows."""
    import torch
    from fasterllama_amd.kv8 import KV8Attention, KV8Cache
    B, H, D, L, T = 2, 1, 128, 128 * 131200, 128  # a slice of 2.15e9 bytes is beyond the limit: see the refusal
    with pytest.raises(capi.FlAttnError):
        KV8Attention(B, H, D, L, torch.float16, T, device=gpu)
    B, L = 33, 128 * 8192  # 33 * 134 MB
    op, cache = KV8Attention(B, H, D, L, torch.float16, T, device=gpu), KV8Cache(B, H, D, L, T, weights=True, device=gpu)
    r = np.random.RandomState(0)
    for b in (0, B - 1):
        cache.k[b, 0, -256:-128] = torch.from_numpy(r.randint(-127, 128, (128, D)).astype(np.int8)).to(gpu)
        cache.v[b, 0, -256:-128] = torch.from_numpy(r.randint(-127, 128, (128, D)).astype(np.int8)).to(gpu)
        cache.k_scale[b, 0, -2], cache.v_scale[b, 0, -2] = 0.03, 0.02
        cache.k_tail[b], cache.v_tail[b] = (torch.from_numpy(r.randn(1, T, D).astype(np.float16)).to(gpu) for _ in range(2))
    mask = torch.full((1, L), NEG, device=gpu)
    mask[:, -256:] = 0
    table = torch.zeros(2, D, device=gpu)
    table[:, 0::2] = 1
    x = [torch.from_numpy(r.randn(B, 1, H, D).astype(np.float16)).to(gpu) for _ in range(3)]
    pos = torch.full((B,), -1, dtype=torch.int32, device=gpu)
    pos[[0, B - 1]] = L - 1
    got = op.decode(*x, cache, table, attn_mask=mask, start_pos_per_seq=pos, max_start_pos=L - 1, rope_row_per_seq=pos * 0)
    torch.cuda.synchronize()
    for b in (0, B - 1):
        small = kr.Cache(1, 1, D, 256, T, seed=1)
        for n in ("k", "v"):
            getattr(small, n)[0, :, :128] = getattr(cache, n)[b, :, -256:-128].cpu().numpy()
            getattr(small, n + "_scale")[0, :, 0] = getattr(cache, n + "_scale")[b, :, -2].cpu().numpy()
            getattr(small, n + "_tail")[0] = getattr(cache, n + "_tail")[b].cpu().numpy()
        want, tol = small.step(*(t[[b]].cpu().numpy() for t in x), table.cpu().numpy(), [255], rope=[0])
        assert_out(got[[b]], want[:, :, 0].reshape(1, D), tol.reshape(1, 1))
        assert np.array_equal(cache.k[b, 0, -128:].cpu().numpy(), small.k[0, 0, 128:])
    assert np.isnan(got[1:B - 1].cpu().numpy()).all()


# ----------------------------------------------------------------------------------------- values of very different sizes

def weighted_tolerance(c, q_rot, P, S, mask):
    """Per query [B,H,S,1], from the reference's state after the call: the 32-bit bound of Cache.tolerance(), relative to what the
    query weighs instead of to the largest |v| of the cache: the larger of max_d sum_j p_j |v_jd| and max_j p_j (absmax of j's block).
    A kernel that holds a weight to 2^-32 of the largest product of weight and block scale adds rows * 2^-32 of the second: 16 U at 4096."""
    ref, T, out = c.ref, c.T, []
    scale = c.scale or 1.0 / math.sqrt(c.D)
    for b in range(c.B):
        k, v = ref.values(b, P + S)
        z = q_rot[b] @ k.transpose(0, 2, 1) * scale
        with np.errstate(invalid="ignore", over="ignore"):
            if mask is not None:
                z = z + mask[P:P + S, :P + S].astype(np.float64)
            e = np.exp(z - np.maximum(z.max(-1, keepdims=True), -1e9))
            p = e / e.sum(-1, keepdims=True)
        n = P + S
        block = np.abs(np.pad(v, ((0, 0), (0, -n % T), (0, 0)))).reshape(c.H, -1, T * c.D).max(-1).repeat(T, -1)[:, :n]
        weighs = np.maximum((p @ np.abs(v)).max(-1), (p * block[:, None]).max(-1))
        A = scale * np.abs(q_rot[b]).max() * np.abs(k).sum(-1).max()
        out.append(kr.U * (4 * A + math.sqrt(n) + 64) * weighs[..., None])
    return np.stack(out)


def prompt_of(c, q, k, v, m, **kw):
    """A prompt of the given float32 inputs [B,S,H,D]: (out, expected, tolerance per query)."""
    P, S = int(c.rows[0]), q.shape[1]
    got = c.op.prefill(c.t(q), c.t(k), c.t(v), c.gpu, c.table_d, start_pos=P, attn_mask=c.t(m), **kw)
    want, _ = c.ref.step(q, k, v, c.table, c.rows, m, None, c.scale)
    return got, want, weighted_tolerance(c, kr.rotate(q, c.table[P:P + S][:, None]).transpose(0, 2, 1, 3), P, S, m)


@pytest.mark.parametrize("kind", [None, "causal"])
@pytest.mark.parametrize("amp", [1.0, 1e-3, 1e-5])
@pytest.mark.parametrize("D,T,S", [(128, 64, 320), (64, 32, 96), (96, 128, 384), (32, 32, 1024), (256, 64, 128)])
def test_values_behind_a_block_of_zeros(gpu, D, T, S, amp, kind):
    """Padding is zeros: a block with no scale says nothing about the size of the values that follow it."""
    c = Case(gpu, 1, 2, D, S + T, T, "f32", 0, max_seq_len=S, weights=D <= 128)
    _, val, _ = c.feed(S, 3)
    q, k, v = (x.copy() for x in val)
    k[:, :T] = 0
    v[:, :T] = 0
    v *= np.float32(amp)
    m = masks(kind, S + T)
    got, want, tol = prompt_of(c, q, k, v, m)
    if kind:
        assert not got[:, :, :T].cpu().numpy().any()  # queries that see zeros only
    assert_out(got, want, tol, f"amp {amp}")
    assert_cache(c.gpu, c.ref, S, S)
    kk, vv = c.op.read(c.gpu, S)
    for x, y in zip((kk, vv), c.ref.values(0, S)):
        assert np.array_equal(x[0].cpu().numpy(), y.astype(np.float32))
    # and a step behind them
    c.rows[:] = S
    _, val, _ = c.feed(1, 4)
    q1, k1, v1 = (x.copy() for x in val)
    v1 *= np.float32(amp)
    got = c.op.decode(c.t(q1), c.t(k1), c.t(v1), c.gpu, c.table_d, start_pos=S)
    want, _ = c.ref.step(q1, k1, v1, c.table, c.rows)
    tol = weighted_tolerance(c, kr.rotate(q1, c.table[S:S + 1][:, None]).transpose(0, 2, 1, 3), S, 1, None)
    assert_out(got, want[:, :, 0], tol[:, :, 0], "step")


@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 14, 2.0 ** 18])
@pytest.mark.parametrize("large", ["first", "last"])
@pytest.mark.parametrize("D,T,start", [(128, 64, 0), (64, 32, 0), (32, 128, 0), (128, 64, 1280)])
def test_large_values_of_little_weight_leave_the_others_precision(gpu, D, T, start, large, ratio):
    """A block of large values with scores 20 lower, before or behind small ones that get nearly all of the weight (`start`: the
    keys are shared by several workgroups)."""
    S = 4 * T if start == 0 else 64
    L = start + S
    c = Case(gpu, 1, 2, D, L, T, "f32", 0, max_seq_len=S if start == 0 else 256)
    _, val, _ = c.feed(L, 5)
    q, k, v = (x.copy() for x in val)
    at = slice(0, T) if large == "first" else slice(L - T, L)
    small = np.ones((1, L, 1, 1), np.float32) / np.float32(ratio)
    small[:, at] = 1
    v *= small
    m = np.zeros((L, L), np.float32)
    m[:, at] = -20
    for P in range(0, start, 256):  # what lies before the piece that is looked at
        n = min(256, start - P)
        c.rows[:] = P
        c.op.prefill(*(c.t(x[:, P:P + n]) for x in (q, k, v)), c.gpu, c.table_d, start_pos=P, attn_mask=c.t(m))
        c.ref.step(*(x[:, P:P + n] for x in (q, k, v)), c.table, c.rows, m)
    c.rows[:] = start
    got, want, tol = prompt_of(c, q[:, start:], k[:, start:], v[:, start:], m)
    assert_out(got, want, tol, f"ratio {ratio}")


@pytest.mark.parametrize("kind", [None, "causal"])
@pytest.mark.parametrize("amp", [1e4, 1e-3, 1e-5])
@pytest.mark.parametrize("D,T,start,S", [(128, 64, 0, 300), (64, 128, 77, 150), (96, 32, 13, 60), (32, 64, 0, 40), (128, 64, 1300, 40), (256, 64, 5, 100)])
def test_small_and_large_values_in_the_open_block(gpu, D, T, start, S, amp, kind):
    """Rows of the open block are values, with no scale beside them; the blocks before them are integers of a scale."""
    L = -(-(start + S) // T) * T
    c = Case(gpu, 1, 2, D, L, T, "f32", 0, max_seq_len=max(S, 256) if L >= 256 else L)
    _, val, _ = c.feed(start + S, 5)
    q, k, v = (x.copy() for x in val)
    v *= np.float32(amp)
    m = masks(kind, L)
    for P in range(0, start, 256):
        n = min(256, start - P)
        c.rows[:] = P
        c.op.prefill(*(c.t(x[:, P:P + n]) for x in (q, k, v)), c.gpu, c.table_d, start_pos=P, attn_mask=c.t(m))
        c.ref.step(*(x[:, P:P + n] for x in (q, k, v)), c.table, c.rows, m)
    c.rows[:] = start
    got, want, tol = prompt_of(c, q[:, start:], k[:, start:], v[:, start:], m)
    assert_out(got, want, tol, f"amp {amp}")
    assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("D,T,start,S", [(128, 64, 0, 320), (64, 32, 77, 150), (96, 128, 0, 300), (32, 32, 0, 64), (128, 64, 1300, 40), (256, 64, 0, 128)])
def test_rows_masked_by_a_finite_value_weigh_their_keys_evenly(gpu, D, T, start, S):
    """-1e9 on every key of a row: next to it a score is less than half a step of a 32-bit float, so all keys weigh the same, as in
    the caches of the other types; the blocks' scales differ."""
    L = -(-(start + S) // T) * T
    c = Case(gpu, 1, 2, D, L, T, "f32", 0, max_seq_len=max(S, 256) if L >= 256 else L)
    _, val, _ = c.feed(start + S, 6)
    q, k, v = (x.copy() for x in val)
    r = np.random.RandomState(0)
    v *= np.exp2(r.randint(-8, 9, (1, -(-(start + S) // T), 1, 1))).astype(np.float32).repeat(T, 1)[:, :start + S]
    m = masks("causal", L)
    m[start + 3:start + 40:3] = -1e9
    for P in range(0, start, 256):
        n = min(256, start - P)
        c.rows[:] = P
        c.op.prefill(*(c.t(x[:, P:P + n]) for x in (q, k, v)), c.gpu, c.table_d, start_pos=P, attn_mask=c.t(m))
        c.ref.step(*(x[:, P:P + n] for x in (q, k, v)), c.table, c.rows, m)
    c.rows[:] = start
    got, want, tol = prompt_of(c, q[:, start:], k[:, start:], v[:, start:], m)
    n = start + S
    _, vv = c.ref.values(0, n)
    for s in range(3, min(S, 40), 3):
        want[0, :, s] = vv.mean(1)
        # n equal weights: the sums' and the quotient's roundings, of the mean |v| (largest over the elements)
        tol[0, :, s] = kr.U * (math.sqrt(n) + 64) * np.abs(vv).mean(1).max(-1, keepdims=True)
    assert_out(got, want, tol)
    # the decode step under such a row
    if n < L:
        c.rows[:] = n
        m[n] = -1e9
        got, want, _ = c.decode(m)
        _, vv = c.ref.values(0, n + 1)
        assert_out(got, vv.mean(1)[None], kr.U * (math.sqrt(n) + 64) * np.abs(vv).mean(1).max(-1)[None, :, None], "step")


# ------------------------------------------------------------------------------------------- long contexts of one workgroup

def long_case(dev, D, T, rows, L, weights=True, **kw):
    """A cache of `rows` rows without the reference's row by row filling: random bytes, neighbouring blocks of different scales."""
    c = Case(dev, 1, 1, D, L, T, "f16", 0, weights=weights, **kw)
    r, n = np.random.RandomState(D + rows), L // T
    c.ref.k_scale[:], c.ref.v_scale[:] = 0.02 * np.exp2(r.randint(-2, 2, (1, 1, n))), 0.02 * np.exp2(r.randint(-3, 3, (1, 1, n)))
    c.ref.k_tail[:], c.ref.v_tail[:] = r.randn(*c.ref.k_tail.shape), r.randn(*c.ref.k_tail.shape)
    if weights:
        c.ref.weights[:] = r.rand(*c.ref.weights.shape)
    c.gpu, c.rows = to_gpu(c.ref, dev), np.array([rows])
    return c


@pytest.mark.parametrize("D,T,rows", [(1024, 32, 1100), (1024, 64, 2111), (1024, 128, 4200), (512, 64, 2200), (256, 32, 4190), (256, 128, 16500),
                                      (128, 64, 8300), (96, 32, 8254), (64, 32, 8319), (32, 128, 8250), (128, 128, 33000)])
@pytest.mark.parametrize("kind", [None, "causal"])
def test_one_workgroup_walks_a_long_context(gpu, D, T, rows, kind):
    """nsplit = 1: more rows than the lanes of a wave hold scales and granules for, and than granules fit beside the merge; two steps,
    of which one may fill a block."""
    L = (rows // T + 2) * T
    c = long_case(gpu, D, T, rows, L, nsplit=1)
    for step in range(2):
        c.rows[:] = rows + step
        m = None
        if kind:  # one row for every position: the last 100 keys and every seventh are hidden
            m = np.zeros((1, L), np.float32)
            m[0, rows - 100:] = NEG
            m[0, ::7] = -np.inf
            m[0, rows:] = 0
        raw, val, _ = c.feed(1, 20 + step)
        got = c.op.decode(*raw, c.gpu, c.table_d, start_pos=rows + step, attn_mask=c.t(m))
        want, tol = c.ref.step(*val, c.table, c.rows, None if m is None else np.broadcast_to(m, (L, L)))
        assert_out(got, want[:, :, 0], tol[..., 0], f"step {step}")
    assert_cache(c.gpu, c.ref, 2)


@pytest.mark.parametrize("D,T,start", [(1024, 32, 1100), (512, 128, 2300), (256, 64, 4200)])
def test_wide_prompt_behind_a_long_context(gpu, D, T, start):
    S, L = 5, (start // T + 2) * T
    c = long_case(gpu, D, T, start, L, weights=False, max_seq_len=S)
    got, want, tol = c.prompt(S, masks("causal", L))
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref, S, start + S)


@pytest.mark.parametrize("D,T", [(256, 64), (1024, 32)])
def test_eviction_where_a_prompt_cannot_gather_weights(gpu, D, T):
    """size_per_head beyond 128: the prompt goes through the same arrays without weights, whose entries the caller zeroes; the steps
    behind it gather, and the eviction goes by them."""
    import torch
    from fasterllama_amd.kv8 import KV8Cache
    L, S = 6 * T, 4 * T + 5
    c = Case(gpu, 2, 2, D, L, T, "f16", 0, weights=True, max_seq_len=S)
    raw, val, _ = c.feed(S, 3)
    with pytest.raises(capi.FlAttnError):
        c.op.prefill(*raw, c.gpu, c.table_d)
    g = c.gpu
    g.weights.zero_()
    c.ref.weights[:] = 0
    c.op.prefill(*raw, KV8Cache.of(T, g.k, g.v, g.k_scale, g.v_scale, g.k_tail, g.v_tail), c.table_d)
    c.ref.step(*val, c.table, c.rows)
    c.ref.weights[:] = 0
    for step in range(3):
        c.rows[:] = S + step
        got, want, tol = c.decode(seed=50 + step)
        assert_out(got, want, tol, f"step {step}")
    assert_cache(c.gpu, c.ref, 3, S + 3)
    c.ref.weights[:] = c.gpu.weights.cpu().numpy()  # (equal but for their last bits, by which close ones would differ)
    kept, after = c.op.evict(c.gpu, 2, 1, S + 3)
    want_kept, _ = kr.evict(c.ref, np.full(2, S + 3), 2, 1)
    assert np.array_equal(kept.cpu().numpy(), want_kept) and (after.cpu().numpy() == 2 * T + 8).all()


@pytest.mark.parametrize("D,T,rows", [(128, 64, 5000), (128, 32, 9000), (32, 128, 17000), (96, 32, 9001), (256, 64, 9000), (1024, 32, 2000)])
@pytest.mark.parametrize("kind", [None, "even"])
@pytest.mark.parametrize("ready", [True, False])
def test_steps_of_many_splits(gpu, D, T, rows, kind, ready):
    """More splits than a merge requests ahead, and more than a wave has lanes; `even`: -1e9 on every key, which then weigh the same."""
    L = (rows // T + 2) * T
    c = long_case(gpu, D, T, rows, L, nsplit=1024)
    if not ready:  # the merge as a launch of its own
        def without(call, *args):
            c.op.io.flags = 0
            capi.check(call(*args, 0))
        c.op._enqueue = without
    import torch
    torch.cuda.synchronize()
    before = c.ref.weights.copy()
    m = np.full((1, L), -1e9, np.float32) if kind else None
    raw, val, _ = c.feed(1, 3)
    got = c.op.decode(*raw, c.gpu, c.table_d, start_pos=rows, attn_mask=c.t(m))
    torch.cuda.synchronize()
    want, tol = c.ref.step(*val, c.table, c.rows)
    want, tol = want[:, :, 0], tol[..., 0]
    if kind:
        n = rows + 1
        _, vv = c.ref.values(0, n)
        want = vv.mean(1)[None]
        tol = kr.U * (math.sqrt(n) + 64) * np.abs(vv).mean(1).max(-1)[None, :, None]
        share = np.minimum(T, n - T * np.arange(-(-n // T))) / n
        c.ref.weights[:, :, :share.size] = np.where(T * np.arange(share.size) >= rows, 0, before[:, :, :share.size]) + share
    assert_out(got, want, tol)
    assert_cache(c.gpu, c.ref)


@pytest.mark.parametrize("D,T", [(64, 32), (128, 32), (512, 64)])
def test_steps_that_fill_a_block_of_zeros(gpu, D, T):
    c = Case(gpu, 1, 2, D, 3 * T, T, "f16", 0, weights=True)
    for step in range(2 * T + 3):
        c.rows[:] = step
        raw, val, _ = c.feed(1, 100 + step)
        q, k, v = (x.copy() for x in val)
        if step < T:
            k[:], v[:] = 0, 0
        got = c.op.decode(c.t(q), c.t(k), c.t(v), c.gpu, c.table_d, start_pos=step)
        want, tol = c.ref.step(q, k, v, c.table, c.rows)
        assert_out(got, want[:, :, 0], tol[..., 0], f"step {step}")
    assert_cache(c.gpu, c.ref, 2 * T + 3)
    assert not c.gpu.k_scale[:, :, 0].cpu().numpy().any() and not c.gpu.k[:, :, :T].cpu().numpy().any()


@pytest.mark.parametrize("D,T,start,S", [(128, 64, 0, 320), (64, 32, 77, 150), (128, 64, 1300, 40)])
def test_block_weights_of_queries_that_weigh_their_keys_evenly(gpu, D, T, start, S):
    L, W = -(-(start + S) // T) * T, 30
    c = Case(gpu, 1, 2, D, L, T, "f16", start, weights=True, max_seq_len=S)
    before, n = c.ref.weights.copy(), start + S
    raw, val, _ = c.feed(S, 4)
    c.op.prefill(*raw, c.gpu, c.table_d, start_pos=start, attn_mask=c.t(np.full((L, L), -1e9, np.float32)), weight_queries=W)
    c.ref.step(*val, c.table, c.rows)
    share = W * np.minimum(T, n - T * np.arange(-(-n // T))) / n
    c.ref.weights[:, :, :share.size] = np.where(T * np.arange(share.size) >= start, 0, before[:, :, :share.size]) + share
    assert_cache(c.gpu, c.ref, W, n)


@pytest.mark.parametrize("bias", [10.0, 30.0, 50.0])
@pytest.mark.parametrize("D,T,S", [(128, 64, 320), (128, 128, 156), (32, 32, 75), (64, 64, 1100), (256, 64, 100)])
def test_zeros_that_take_the_weight(gpu, D, T, S, bias):
    """A block of zeros with scores `bias` higher: next to nothing is left for the others, and all of the output comes from it."""
    L = -(-S // T) * T
    c = Case(gpu, 1, 2, D, L, T, "f32", 0, max_seq_len=S, weights=D <= 128)
    _, val, _ = c.feed(S, 3)
    q, k, v = (x.copy() for x in val)
    v[:, :T] = 0
    m = np.full((1, L), -bias, np.float32)
    m[:, :T] = 0
    m = np.broadcast_to(m, (L, L))
    got, want, tol = prompt_of(c, q, k, v, m)
    # beside the products' errors, a score rounds next to a mask entry of `bias`, before and after the change of base: 4 U of it
    assert_out(got, want, tol * (1 + 4 * bias / 64), f"bias {bias}")
    assert_cache(c.gpu, c.ref, S, S)
