"""Host logic of the 8-bit cache's calls: struct sizes, refusals, workspace sizes.  No kernel is launched: every call here is
rejected before a launch."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from fasterllama_amd import build, capi


def desc(B=2, H=4, D=128, L=256, dtype=capi.FL_ATTN_F16, nsplit=0, scale=0.0, flags=0):
    return capi.AttnDesc(B, H, D, L, dtype, nsplit, scale, flags)


def fake_cache(block_len=64, weights=0x900000, at=0x1000000, **over):
    c = capi.Kv8CacheArrays(block_len=block_len, k=at, v=at + 0x100000, k_scale=at + 0x200000, v_scale=at + 0x300000,
                            k_tail=at + 0x400000, v_tail=at + 0x500000, weights=weights)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def fake_io(**over):
    io = capi.AttnIO()
    for name in ("q", "k_new", "v_new", "freq_cis", "out"):
        setattr(io, name, 0x1000)
    io.workspace, io.workspace_bytes = 0x10000, 1 << 40
    io.mask_ld, io.start_pos, io.rope_row, io.max_start_pos = 256, 3, -1, -1
    for k, v in over.items():
        setattr(io, k, v)
    return io


def decode(d=None, c=None, io=None, rope=None, rows=64):
    return capi.load().fl_kv8_decode_forward(C.byref(d or desc()), C.byref(c or fake_cache()), C.byref(io or fake_io()), rope, rows, None)


def prefill(d=None, c=None, io=None, S=8, W=0, lens=None):
    return capi.load().fl_kv8_prefill_forward(C.byref(d or desc()), C.byref(c or fake_cache()), C.byref(io or fake_io()), S, lens, W, None)


def evict(d=None, c=None, to=None, **over):
    kw = dict(rows=200, keep_blocks=2, recent_blocks=1, kept=0x20000, rows_out=0x30000)
    kw.update(over)
    args = capi.Kv8EvictArgs(**kw)
    args.struct_size = kw.get("struct_size", args.struct_size)
    c = c or fake_cache()
    return capi.load().fl_kv8_evict(C.byref(d or desc()), C.byref(c), C.byref(to or c), C.byref(args), None)


def test_struct_layouts():
    assert C.sizeof(capi.Kv8CacheArrays) == 8 + 7 * 8
    assert C.sizeof(capi.Kv8EvictArgs) == 8 + 8 + 4 * 4 + 2 * 8


@pytest.mark.parametrize("kw,want", [
    (dict(D=48), capi.FL_ATTN_ERR_HEAD_DIM), (dict(B=0), capi.FL_ATTN_ERR_SHAPE), (dict(dtype=2), capi.FL_ATTN_ERR_DTYPE),
    (dict(L=250), capi.FL_ATTN_ERR_SHAPE),          # not a multiple of the block
    (dict(nsplit=5000), capi.FL_ATTN_ERR_ARGUMENT), (dict(scale=float("nan")), capi.FL_ATTN_ERR_ARGUMENT),
])
def test_descriptor(kw, want):
    d, n = desc(**kw), C.c_size_t()
    lib = capi.load()
    assert lib.fl_kv8_workspace_bytes(C.byref(d), 64, 1, C.byref(n)) == want
    assert lib.fl_kv8_workspace_init(C.byref(d), 64, 1, 0x10000, 1 << 40, None) == want
    assert lib.fl_kv8_cache_bytes(C.byref(d), 64, C.byref(n), C.byref(n), C.byref(n)) == want
    assert decode(d) == want and prefill(d) == want and evict(d) == want
    assert lib.fl_kv8_read(C.byref(d), C.byref(fake_cache()), 8, None, 0x1000, 0x2000, None) == want


@pytest.mark.parametrize("over,want", [
    (dict(block_len=0), capi.FL_ATTN_ERR_SHAPE), (dict(block_len=48), capi.FL_ATTN_ERR_SHAPE), (dict(block_len=256), capi.FL_ATTN_ERR_SHAPE),
    (dict(struct_size=0), capi.FL_ATTN_ERR_STRUCT_SIZE), (dict(struct_size=72), capi.FL_ATTN_ERR_STRUCT_SIZE),
    *[({n: None}, capi.FL_ATTN_ERR_NULL_POINTER) for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")],
    *[({n: 0x1000008}, capi.FL_ATTN_ERR_ALIGNMENT) for n in ("k", "v", "k_tail", "v_tail")],
    *[({n: 0x1000002}, capi.FL_ATTN_ERR_ALIGNMENT) for n in ("k_scale", "v_scale", "weights")],
])
def test_cache(over, want):
    c = fake_cache(**over)
    assert decode(c=c) == want and prefill(c=c) == want and evict(c=c) == want
    assert capi.load().fl_kv8_read(C.byref(desc()), C.byref(c), 8, None, 0x1000, 0x2000, None) == want


@pytest.mark.parametrize("over,want", [
    *[({n: None}, capi.FL_ATTN_ERR_NULL_POINTER) for n in ("q", "k_new", "v_new", "freq_cis", "out")],
    *[({n: 0x1004}, capi.FL_ATTN_ERR_ALIGNMENT) for n in ("q", "k_new", "v_new", "freq_cis", "out")],
    (dict(out_int8=0x1000), capi.FL_ATTN_ERR_NULL_POINTER), (dict(out_int8=0x1001, out_scale=0x1000), capi.FL_ATTN_ERR_ALIGNMENT),
    (dict(qkv_inp_scale=0x1000), capi.FL_ATTN_ERR_NULL_POINTER), (dict(q_weight_scale=0x1000), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(start_pos=-1), capi.FL_ATTN_ERR_POSITION), (dict(start_pos=256), capi.FL_ATTN_ERR_POSITION),
    (dict(rope_row=-2), capi.FL_ATTN_ERR_POSITION), (dict(flags=2), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(attn_mask=0x1000, mask_ld=3), capi.FL_ATTN_ERR_ARGUMENT), (dict(attn_mask=0x1000, mask_ld=-1), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(workspace=None), capi.FL_ATTN_ERR_WORKSPACE), (dict(workspace=0x10080), capi.FL_ATTN_ERR_WORKSPACE),
    (dict(workspace_bytes=64), capi.FL_ATTN_ERR_WORKSPACE), (dict(struct_size=8), capi.FL_ATTN_ERR_STRUCT_SIZE),
])
def test_io(over, want):
    assert decode(io=fake_io(**over)) == want
    assert prefill(io=fake_io(**over)) == want


def test_decode_only_and_prompt_only():
    assert decode(rope=0x1002) == capi.FL_ATTN_ERR_ALIGNMENT
    assert decode(rope=0x1000, rows=0) == capi.FL_ATTN_ERR_POSITION
    assert decode(io=fake_io(start_pos_per_seq=0x1000, max_start_pos=256)) == capi.FL_ATTN_ERR_POSITION
    assert prefill(io=fake_io(start_pos_per_seq=0x1000)) == capi.FL_ATTN_ERR_ARGUMENT
    assert prefill(S=0) == capi.FL_ATTN_ERR_POSITION and prefill(S=254) == capi.FL_ATTN_ERR_POSITION
    assert prefill(W=-1) == capi.FL_ATTN_ERR_ARGUMENT
    assert prefill(lens=0x1002) == capi.FL_ATTN_ERR_ALIGNMENT
    assert prefill(d=desc(D=256)) == capi.FL_ATTN_ERR_HEAD_DIM  # weights beyond 128
    wide = desc(B=64, H=64, D=256, L=8192)  # a workgroup per query: 2^32 threads
    assert prefill(d=wide, c=fake_cache(weights=None), io=fake_io(start_pos=0), S=4096) == capi.FL_ATTN_ERR_SHAPE
    many = desc(B=1024, H=64, D=32, L=8192)  # blocks to fill
    assert prefill(d=many, c=fake_cache(weights=None), io=fake_io(start_pos=0), S=8192) == capi.FL_ATTN_ERR_SHAPE
    tokens = desc(B=4096, H=1, D=32, L=4096)  # tokens to quantise
    io = fake_io(start_pos=0, out_int8=0x1000, out_scale=0x1000)
    assert prefill(d=tokens, c=fake_cache(weights=None), io=io, S=4096) == capi.FL_ATTN_ERR_SHAPE
    n = C.c_size_t()
    assert capi.load().fl_kv8_workspace_bytes(C.byref(desc()), 64, 257, C.byref(n)) == capi.FL_ATTN_ERR_POSITION


def test_read_refusals():
    lib, d, c = capi.load(), desc(), fake_cache()
    for rows, k, v, per, want in ((0, 0x1000, 0x2000, None, capi.FL_ATTN_ERR_POSITION), (257, 0x1000, 0x2000, None, capi.FL_ATTN_ERR_POSITION),
                                  (8, None, 0x2000, None, capi.FL_ATTN_ERR_NULL_POINTER), (8, 0x1000, 0x2008, None, capi.FL_ATTN_ERR_ALIGNMENT),
                                  (8, 0x1000, 0x2000, 0x3001, capi.FL_ATTN_ERR_ALIGNMENT)):
        assert lib.fl_kv8_read(C.byref(d), C.byref(c), rows, per, k, v, None) == want


@pytest.mark.parametrize("over,want", [
    (dict(keep_blocks=0), capi.FL_ATTN_ERR_ARGUMENT), (dict(keep_blocks=5), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(recent_blocks=-1), capi.FL_ATTN_ERR_ARGUMENT), (dict(recent_blocks=3), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(rows=-1), capi.FL_ATTN_ERR_POSITION), (dict(rows=257), capi.FL_ATTN_ERR_POSITION),
    (dict(kept=None), capi.FL_ATTN_ERR_NULL_POINTER), (dict(rows_out=None), capi.FL_ATTN_ERR_NULL_POINTER),
    (dict(kept=0x1002), capi.FL_ATTN_ERR_ALIGNMENT), (dict(rows_per_seq=0x1002), capi.FL_ATTN_ERR_ALIGNMENT),
    (dict(to_total_len=-64), capi.FL_ATTN_ERR_ARGUMENT), (dict(to_total_len=100), capi.FL_ATTN_ERR_SHAPE),
    (dict(to_total_len=128), capi.FL_ATTN_ERR_ARGUMENT),   # in place, another length
    (dict(rows_per_seq=0x30004), capi.FL_ATTN_ERR_ARGUMENT), (dict(rows_per_seq=0x2003c), capi.FL_ATTN_ERR_ARGUMENT),  # written ranges
    (dict(rows_out=0x2003c), capi.FL_ATTN_ERR_ARGUMENT),
    (dict(reserved=1), capi.FL_ATTN_ERR_ARGUMENT), (dict(struct_size=16), capi.FL_ATTN_ERR_STRUCT_SIZE),
])
def test_evict_refusals(over, want):
    assert evict(**over) == want


def test_evict_refuses_caches_that_overlap_in_part():
    bh, rows = 8, 8 * 256 * 128
    a = fake_cache()
    for name, shift in (("k", 4096), ("v", -4096), ("k_scale", 16), ("v_scale", 4), ("weights", 8), ("k_tail", 32), ("v_tail", 64)):
        b = fake_cache(at=0x8000000, weights=0xa00000)
        setattr(b, name, getattr(a, name) + shift)
        assert evict(c=a, to=b) == capi.FL_ATTN_ERR_ARGUMENT, name
    b = fake_cache(at=0x8000000, weights=0xa00000)
    b.k = a.v + rows - 16           # another array's end
    assert evict(c=a, to=b) == capi.FL_ATTN_ERR_ARGUMENT
    b = fake_cache(at=0x8000000, weights=0xa00000)
    b.k = a.k                       # the same in part
    assert evict(c=a, to=b) == capi.FL_ATTN_ERR_ARGUMENT
    assert evict(c=a, to=fake_cache(block_len=32, at=0x8000000, weights=0xa00000)) == capi.FL_ATTN_ERR_ARGUMENT
    assert evict(c=fake_cache(weights=None)) == capi.FL_ATTN_ERR_NULL_POINTER


def test_cache_bytes_and_workspace_sizes():
    lib = capi.load()
    r, s, t, n, m = (C.c_size_t() for _ in range(5))
    assert lib.fl_kv8_cache_bytes(C.byref(desc(B=64, H=32, D=128, L=8192)), 64, C.byref(r), C.byref(s), C.byref(t)) == 0
    assert (r.value, s.value, t.value) == (64 * 32 * 8192 * 128, 64 * 32 * 128 * 4, 64 * 32 * 64 * 128 * 2)
    for D in (32, 64, 96, 128, 256, 512, 1024):
        d = desc(D=D, L=1024, nsplit=7)
        assert lib.fl_kv8_workspace_bytes(C.byref(d), 32, 1, C.byref(n)) == 0
        assert lib.fl_kv8_workspace_bytes(C.byref(d), 32, 500, C.byref(m)) == 0
        assert n.value % 256 == 0 and m.value >= n.value >= 8 * (4 + D * 4 + 7 * (D + 2) * 4 + 1024 // 32 * 8)
    # a workspace for prompts of up to S tokens serves every shorter one
    for B, H, D in ((1, 4, 128), (3, 43, 96), (1, 129, 32), (2, 128, 64), (1, 257, 128), (1, 8, 256)):
        d, last = desc(B=B, H=H, D=D, L=1024), 0
        for S in (1, 2, 31, 32, 33, 127, 128, 129, 256, 257, 512, 1024):
            assert lib.fl_kv8_workspace_bytes(C.byref(d), 64, S, C.byref(n)) == 0 and n.value >= last
            last = n.value
    assert lib.fl_kv8_workspace_bytes(C.byref(desc()), 64, 1, None) == capi.FL_ATTN_ERR_NULL_POINTER


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_no_kernel_spills_registers(tmp_path):
    flags = [f for f in build.HIP_FLAGS if f != "-fPIC"]
    res = subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-c", "-Rpass-analysis=kernel-resource-usage", "-o", str(tmp_path / "x.o"),
                          os.path.join(build.CSRC, "fl_kv8.hip")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout[-2000:]
    name, seen, bad = None, 0, []
    for line in res.stdout.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            name, seen = m.group(1), seen + 1
        m = re.search(r"(ScratchSize \[bytes/lane\]|VGPRs Spill): (\d+)", line)
        if m and int(m.group(2)) > 0:
            bad.append((name, m.group(1), int(m.group(2))))
    assert seen > 40 and not bad, (seen, bad)
