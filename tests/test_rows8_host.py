"""Rows held in 8 bits: layout and refusals that need no GPU."""

import pytest
import torch


@pytest.mark.parametrize("d,want", [(1, 48), (31, 48), (32, 48), (33, 80), (64, 80), (768, 800), (1037, 1104), (4096, 4224)])
def test_pitch(pkg, d, want):
    assert pkg.ops.rows8_pitch(d) == want == pkg._lib.load().sae_rows8_pitch(d)


def test_pitch_of_nothing(pkg):
    lib = pkg._lib.load()
    assert lib.sae_rows8_pitch(0) == 0 and lib.sae_rows8_pitch(-4) == 0


@pytest.mark.parametrize("tokens", [1, 64, 100, 4096, 131072])
@pytest.mark.parametrize("m,n", [(1, 1), (64, 64), (1003, 521), (8192, 2048)])
@pytest.mark.parametrize("wide", [False, True])
def test_a_slice_holds_a_slab(pkg, tokens, m, n, wide):
    s = pkg.ops._over_tokens_slices(tokens, m, n, wide)
    assert 1 <= s <= -(-tokens // (32 if wide else 64))


@pytest.mark.parametrize("tokens,m,n", [(32768, 2048, 2048), (131072, 32768, 2048), (8192, 4096, 2048), (16384, 4096, 4096), (65536, 8192, 8192)])
@pytest.mark.parametrize("wide", [False, True])
def test_a_full_card_is_not_cut(pkg, tokens, m, n, wide):
    """Whole rounds of the four workgroups that each of 256 CUs holds: slices would take partial results and save nothing."""
    assert -(-m // 64) * -(-n // 64) % 1024 == 0 and pkg.ops._over_tokens_slices(tokens, m, n, wide) == 1


def test_rows8_holds_whole_records(pkg):
    R = pkg.Rows8
    ok = R(torch.zeros(3, 80, dtype=torch.uint8), 40)
    assert ok.shape == (3, 40) and len(ok) == 3 and ok.device.type == "cpu"
    for data, d in [(torch.zeros(3, 80), 40), (torch.zeros(3, 96, dtype=torch.uint8), 40), (torch.zeros(80, dtype=torch.uint8), 40),
                    (torch.zeros(3, 48, dtype=torch.uint8), 40), (torch.zeros(3, 0, dtype=torch.uint8), 0)]:
        with pytest.raises(ValueError):
            R(data, d)


def test_rows8_stay_what_they_were_made(pkg):
    """The kernels read records by the width they were made with."""
    q = pkg.Rows8(torch.zeros(3, pkg.ops.rows8_pitch(40), dtype=torch.uint8), 40)
    for name, value in (("data", q.data[:, :32]), ("d", 41)):
        with pytest.raises(AttributeError):
            setattr(q, name, value)


def test_an_index_is_of_32_bit_entries_side_by_side(pkg):
    """The kernels read it by its addresses: wider entries, or entries that lie apart, would be read as slots and tokens that do not
    exist."""
    ptr, slot, tok = (torch.zeros(n, dtype=torch.int32) for n in (5, 8, 8))
    fi = pkg.FeatureIndex(ptr, slot, tok)
    for i in range(3):
        for wrong in (torch.int64, torch.int16, torch.float32):
            with pytest.raises(TypeError):
                pkg.FeatureIndex(*[t.to(wrong) if j == i else t for j, t in enumerate((ptr, slot, tok))])
        for wrong in (lambda t: torch.stack([t, t], 1)[:, 0], lambda t: t[None], lambda t: t[:1].expand(len(t))):
            with pytest.raises(ValueError):
                pkg.FeatureIndex(*[wrong(t) if j == i else t for j, t in enumerate((ptr, slot, tok))])
    assert pkg.FeatureIndex(ptr[1:4], slot, tok).feat_ptr.numel() == 3
    for name in ("feat_ptr", "feat_slot", "slot_tok"):
        with pytest.raises(AttributeError):
            setattr(fi, name, tok.long())


def test_every_slot_has_a_coefficient(pkg):
    fi = pkg.FeatureIndex(*(torch.zeros(n, dtype=torch.int32) for n in (5, 8, 8)))
    pkg.ops._req_slots(fi, torch.zeros(8))
    with pytest.raises(ValueError, match="7 coefficients"):
        pkg.ops._req_slots(fi, torch.zeros(7))


def test_the_kernels_have_no_cpu_fallback(pkg):
    ops = pkg.ops
    q = ops.Rows8(torch.zeros(3, 80, dtype=torch.uint8), 40)
    with pytest.raises(RuntimeError):
        ops.quantize_rows(torch.zeros(3, 40))
    with pytest.raises(RuntimeError):
        ops.restore_rows(q)
    with pytest.raises(RuntimeError):
        ops.gather_rows(q, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.gemm_over_tokens(torch.zeros(3, 8, dtype=torch.bfloat16), q)


def test_entry_points_refuse_before_any_launch(pkg):
    """Null pointers, sizes, types, alignment: rejected on the host (the pointers below are never read)."""
    lib = pkg._lib.load()
    P = 1 << 20
    quant = lambda src=P, dt=0, n=4, d=40, stride=40, rows=P, copy=None: lib.sae_rows8_quantize(src, dt, n, d, stride, rows, copy, None)  # noqa: E731
    assert quant(src=None) == -1 and quant(rows=None) == -1 and quant(n=0) == -1 and quant(d=0) == -1 and quant(stride=-1) == -1
    assert quant(dt=2) == -1 and quant(dt=1, copy=P) == -1 and quant(rows=P + 8) == -1 and quant(n=1 << 31) == -2 and quant(d=1 << 30) == -2
    gather = lambda rows=P, idx=P, ns=4, n=4, d=40, dst=P, dt=0: lib.sae_rows8_gather(rows, idx, ns, n, d, dst, dt, 1.0, None)  # noqa: E731
    assert gather(rows=None) == -1 and gather(dst=None) == -1 and gather(ns=0) == -1 and gather(n=0) == -1 and gather(d=-1) == -1
    assert gather(idx=None, n=5) == -1 and gather(dt=2) == -1 and gather(rows=P + 1) == -1 and gather(n=1 << 31) == -2
    tr = lambda src=P, dt=2, r=4, c=40, dst=P, pitch=64: lib.sae_transpose_padded(src, dt, r, c, dst, pitch, None)  # noqa: E731
    assert tr(src=None) == -1 and tr(dst=None) == -1 and tr(r=0) == -1 and tr(pitch=3) == -1 and tr(pitch=60) == -1 and tr(dt=0) == -1
    assert tr(dst=P + 2) == -1 and tr(src=P + 8) == -1 and tr(pitch=1 << 30) == -2
    ot = lambda l=P, ldt=1, r=P, rdt=2, T=100, m=8, n=8, out=P, odt=0, s=1, part=None: lib.sae_gemm_over_tokens(  # noqa: E731
        l, ldt, r, rdt, T, m, n, out, odt, s, part, None)
    assert ot(l=None) == -1 and ot(r=None) == -1 and ot(out=None) == -1 and ot(T=0) == -1 and ot(m=0) == -1 and ot(n=-1) == -1
    assert ot(ldt=3) == -1 and ot(rdt=-1) == -1 and ot(odt=2) == -1 and ot(ldt=0, odt=1) == -1 and ot(r=P + 8) == -1
    assert ot(s=0) == -1 and ot(s=2) == -1 and ot(s=3, part=P) == -1 and ot(n=65535 * 64 + 1) == -2 and ot(m=1 << 29) == -2
    join = lambda p=P, s=2, c=100, out=P, odt=0: lib.sae_join_slices(p, s, c, out, odt, None)   # noqa: E731
    assert join(p=None) == -1 and join(out=None) == -1 and join(s=0) == -1 and join(c=0) == -1 and join(odt=2) == -1 and join(c=1 << 42) == -2
    need = lib.sae_rows8_grad_rows_workspace_bytes(2000, 100, 4, 40)
    assert need >= 100 * 4 and lib.sae_rows8_grad_rows_workspace_bytes(2000, 0, 4, 40) == 0
    assert lib.sae_rows8_grad_rows_workspace_bytes(1024, 100, 4, 40) == 0 < lib.sae_rows8_grad_rows_workspace_bytes(1024, 129, 4, 40)   # one launch
    rows = lambda r=P, nr=2000, out=P, F=4, d=40, n=100, ws=P, b=need: lib.sae_rows8_grad_rows(  # noqa: E731
        P, P, P, P, r, nr, out, None, F, d, n, ws, b, None)
    assert rows(nr=0) == -1 and rows(r=None) == -1 and rows(out=None) == -1 and rows(F=0) == -1 and rows(d=0) == -1 and rows(n=0) == -1
    assert rows(r=P + 8) == -1 and rows(ws=None) == -4 and rows(b=need - 1) == -4 and rows(d=65535 * 256 + 4, b=1 << 60) == -2 and rows(out=P + 4) == -1 and rows(out=P + 2, d=41) == -1 and rows(n=(1 << 31) - 1) == -2
    assert lib.sae_sparse_grad_rows(P, P, P, P, P, 2, P, None, 4, 40, None) == -1      # records have their own entry point


def test_launches_that_one_grid_cannot_hold_are_refused(pkg):
    """A grid's first axis counts less than 2^32 threads: larger calls are refused before the first launch, not by the last."""
    lib = pkg._lib.load()
    P = 1 << 20

    def rows(nr, F, d, n):
        return lib.sae_rows8_grad_rows(P, P, P, P, P, nr, P, None, F, d, n, P, 1 << 62, None)

    assert rows(100, (1 << 26) + 1, 1, 10) == -2                     # one launch, eight features a workgroup of 512
    assert rows(4096, (1 << 26) + 1, 1, 10) == -2                    # the first of three, four features a workgroup of 256
    assert rows(4096, (1 << 26) - 8, 1, 1 << 30) == -2               # features and positions together
    assert rows(4096, 1000, 4096, (1 << 29) + 1) == -2               # the second: a wave per window and 256 columns
    assert rows(4096, 1000, 260, (1 << 30) + 1) == -2                # the third: 512 threads per window
    join = lambda count, s=2: lib.sae_join_slices(P, s, count, P, 0, None)   # noqa: E731
    assert join((1 << 34) - 1023) == -2
    ot = lambda m, n, s: lib.sae_gemm_over_tokens(P, 1, P, 1, 640, m, n, P, 0, s, P, None)   # noqa: E731
    assert ot(1 << 20, 1 << 14, 2) == -2


@pytest.mark.parametrize("T,k,d,length", [(1100, 32, 512, 32), (2048, 32, 768, 64), (4096, 32, 768, 64), (4096, 64, 768, 128), (8192, 32, 768, 128),
                                          (8192, 64, 2048, 128)])
def test_windows_are_those_measured_best(pkg, T, k, d, length):
    """Seen by the workspace: feature, token and coefficient of every position, two partial rows per window."""
    windows = -(-T * k // length)
    want = windows * (length * 12 + 2 * -(-d // 32) * 32 * 4)
    assert pkg._lib.load().sae_rows8_grad_rows_workspace_bytes(T, T * k, 8192, d) == want


# ---- records made and read without a GPU; the pipeline that carries them -----------------------------------------------

def exact_values(x):
    """[n, d] fp64: what 8 bits hold of x, block by block, from the definition."""
    import numpy as np

    x = x.double().numpy()
    out = np.zeros_like(x)
    for i in range(x.shape[0]):
        for b in range(0, x.shape[1], 32):
            block = x[i, b : b + 32]
            if not np.isfinite(block).all():
                out[i, b : b + 32] = np.nan
                continue
            top = np.abs(block).max()
            if top == 0:
                continue
            k = max(int(np.floor(np.log2(top))) - 6, -126)
            k += np.rint(np.ldexp(top, -k)) > 127 and k < 121
            out[i, b : b + 32] = np.ldexp(np.clip(np.rint(np.ldexp(block, -k)), -127, 127), k)
    return torch.from_numpy(out)


def rows(n, d, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, d, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 32), (7, 33), (4, 100), (3, 768)])
def test_pack_and_unpack_on_the_cpu(pkg, n, d, dtype):
    x = rows(n, d, 1, dtype)
    data = pkg.rows8_pack(x)
    assert data.dtype == torch.uint8 and tuple(data.shape) == (n, pkg.ops.rows8_pitch(d))
    assert not data[:, 33 * (-(-d // 32)):].any()
    back = pkg.rows8_unpack(data, d, torch.float32)
    assert torch.equal(back.double(), exact_values(x))
    assert torch.equal(pkg.rows8_unpack(data, d, torch.bfloat16).float(), back)
    assert torch.equal(pkg.rows8_unpack(data, d, torch.float32, 0.3), back * 0.3)
    assert torch.equal(pkg.rows8_pack(back), data) or torch.equal(pkg.rows8_unpack(pkg.rows8_pack(back), d, torch.float32), back)
    stacked = pkg.rows8_pack(x.view(1, n, d))
    assert tuple(stacked.shape) == (1, n, data.shape[1]) and torch.equal(stacked[0], data)
    assert torch.equal(pkg.rows8_unpack(stacked, d, torch.float32)[0], back)


def test_pack_extremes_on_the_cpu(pkg):
    top = torch.finfo(torch.float32).max
    x = torch.zeros(10, 64)
    x[:, 0] = torch.tensor([float("inf"), float("nan"), top, -top, 2.0**-126, 1e-44, 0.0, -0.0, 127.5 / 64, 2.0**-121])
    x[:, 40] = 1.0
    back = pkg.rows8_unpack(pkg.rows8_pack(x), 64, torch.float32)
    assert back[:2, :32].isnan().all() and torch.isfinite(back[2:]).all() and (back[:, 40] == 1).all()
    assert torch.equal(back[2:].double(), exact_values(x[2:]))


@pytest.mark.parametrize("shape", [(0, 40), (2, 0, 33), (0, 5, 32), (0, 1)])
def test_no_rows_on_the_cpu(pkg, shape):
    data = pkg.rows8_pack(torch.zeros(shape))
    assert data.dtype == torch.uint8 and tuple(data.shape) == (*shape[:-1], pkg.ops.rows8_pitch(shape[-1]))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        back = pkg.rows8_unpack(data, shape[-1], dtype, 0.5)
        assert back.dtype == dtype and tuple(back.shape) == shape


def test_pack_refuses_other_rows(pkg):
    for bad in (torch.zeros(3, 4, dtype=torch.float64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            pkg.rows8_pack(bad)
    with pytest.raises(ValueError):
        pkg.rows8_unpack(torch.zeros(3, 48, dtype=torch.uint8), 40, torch.float32)


def samples(n, ctx, d, dtype=torch.float32):
    for i in range(n):
        t = torch.arange(ctx)[None] + 100 * i
        yield {"h0": rows(ctx, d, 10 + i, dtype)[None], "h1": rows(ctx, d + 3, 50 + i, dtype)[None], "tokens": t,
               "mask": (t % 5 != 0).to(torch.int64), "attention_mask": torch.ones_like(t), "meta": {"i": i}}


@pytest.mark.parametrize("fmt", ["safetensors", "pt"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_written_and_loaded(pkg, tmp_path, fmt, dtype):
    hooks = ["h0", "h1"]
    pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path / "q"), hook_points=hooks, n_samples_per_chunk=2, format=fmt,
                                                    row_format="rows8")).process(samples(5, 9, 70, dtype))
    pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path / "f"), hook_points=hooks, n_samples_per_chunk=2, format=fmt)
                         ).process(samples(5, 9, 70, dtype))
    dirs = lambda k: {hp: tmp_path / k / hp for hp in hooks}  # noqa: E731
    floats = list(pkg.CachedActivationLoader(dirs("f")).process())
    loader = pkg.CachedActivationLoader(dirs("q"))
    got = list(loader.process())
    kept_loader = pkg.CachedActivationLoader(dirs("q"), keep_rows8=True)
    kept = list(kept_loader.process())
    wide = list(pkg.CachedActivationLoader(dirs("q"), dtype=torch.float32).process())
    assert len(got) == len(floats) == 3 and kept_loader.rows8_widths == {"h0": 70, "h1": 73}
    for a, b, c, w in zip(got, floats, kept, wide):
        assert torch.equal(a["tokens"], b["tokens"]) and a["meta"] == b["meta"]
        for hp, d in (("h0", 70), ("h1", 73)):
            want = exact_values(b[hp].reshape(-1, d)).view(b[hp].shape)
            assert a[hp].dtype == dtype and w[hp].dtype == torch.float32 and torch.equal(w[hp].double(), want)
            assert torch.equal(a[hp], want.to(dtype))
            assert c[hp].dtype == torch.uint8 and tuple(c[hp].shape) == (*b[hp].shape[:-1], pkg.ops.rows8_pitch(d))


def test_stream_of_records_gives_the_rows_they_hold(pkg, tmp_path):
    """Shuffled batches out of a buffer of records = the same draws out of a buffer of the values."""
    hooks = ["h0", "h1"]
    pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path), hook_points=hooks, n_samples_per_chunk=2, row_format="rows8")
                         ).process(samples(7, 12, 70))
    kw = dict(batch_size=10, buffer_size=30, buffer_shuffle_config=pkg.BufferShuffleConfig(perm_seed=3), device="cpu")
    plain = list(pkg.cached_activation_stream(tmp_path, hooks, **kw))
    held = list(pkg.cached_activation_stream(tmp_path, hooks, rows8=True, **kw))
    low = list(pkg.cached_activation_stream(tmp_path, hooks, rows8=True, dtype=torch.float32, **kw))
    over = list(pkg.cached_activation_stream(tmp_path, hooks, rows8=True, override_dtype=torch.float16, **kw))
    assert len(plain) == len(held) == len(low) == len(over) > 4
    for a, b, c, o in zip(plain, held, low, over):
        assert torch.equal(a["tokens"], b["tokens"])
        for hp in hooks:
            assert b[hp].dtype == torch.bfloat16 and c[hp].dtype == torch.float32 and o[hp].dtype == torch.float16
            assert torch.equal(b[hp].float(), a[hp]) and torch.equal(c[hp], a[hp]) and torch.equal(o[hp], a[hp].half())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, None])
def test_a_stream_of_floats_holds_floats(pkg, tmp_path, dtype):
    """Unless records are asked for, nothing rounds the loader's floats to 8 bits again: fp16 values past its largest stay
    infinities by themselves, and rows of a float file in front of 8-bit ones stay what they are."""
    want = torch.cat([w.reshape(-1, 40) for w in write_chunks(pkg, tmp_path, [(40, torch.float32, "float"), (40, torch.float32, "rows8")])])
    want = want.to(dtype) if dtype is not None else want
    got = list(pkg.cached_activation_stream(tmp_path, ["h0"], batch_size=5, buffer_size=10, device="cpu", dtype=dtype))
    assert len(got) > 1 and all(b["h0"].dtype == want.dtype for b in got)
    got = torch.cat([b["h0"] for b in got])
    kept = torch.cat([c["mask"].reshape(-1) for c in pkg.CachedActivationLoader({"h0": tmp_path / "h0"}).process()]).bool()
    assert not got.isnan().any() and torch.equal(got.sort(0).values, want[kept].sort(0).values)
    if dtype == torch.float16:
        assert int(got.isinf().sum()) == int(want[kept].isinf().sum())


def test_a_float_stream_of_records_is_not_rounded_again(pkg, tmp_path):
    """The same over 8-bit files alone: the floats of the records, cast."""
    part = list(samples(2, 4, 40, torch.float32))
    part[0]["h0"][0, 1, 3] = 1e5
    pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path), hook_points=["h0"], n_samples_per_chunk=2, row_format="rows8")
                         ).process(part)
    (chunk,) = pkg.CachedActivationLoader({"h0": tmp_path / "h0"}, dtype=torch.float16).process()
    want = chunk["h0"].reshape(-1, 40)[chunk["mask"].reshape(-1).bool()]
    assert int(want.isinf().sum()) == 1
    got = torch.cat([b["h0"] for b in pkg.cached_activation_stream(tmp_path, ["h0"], batch_size=5, buffer_size=10, device="cpu",
                                                                   dtype=torch.float16)])
    assert not got.isnan().any() and torch.equal(got.sort(0).values, want.sort(0).values)


def test_buffer_that_quantises_what_arrives(pkg):
    data = [{"x": rows(n, 45, n), "y": torch.arange(n)} for n in (7, 20, 3, 31)]
    kw = dict(buffer_size=24, buffer_shuffle_config=pkg.BufferShuffleConfig(perm_seed=1))
    plain = list(pkg.ActivationBatchler(6, **kw).process(data))
    held = list(pkg.ActivationBatchler(6, rows8={"x": 45}, **kw).process(data))
    scaled = list(pkg.ActivationBatchler(6, rows8={"x": 45}, scale=0.5, override_dtype=torch.bfloat16, **kw).process(data))
    assert len(plain) == len(held) == len(scaled)
    for a, b, c in zip(plain, held, scaled):
        want = exact_values(a["x"])
        assert torch.equal(a["y"], b["y"]) and b["x"].dtype == torch.float32 and torch.equal(b["x"].double(), want)
        assert c["x"].dtype == torch.bfloat16 and torch.equal(c["x"], (want * 0.5).to(torch.bfloat16))
    mixed = [data[0], {"x": pkg.rows8_pack(data[1]["x"]), "y": data[1]["y"]}]
    out = torch.cat([b["x"] for b in pkg.ActivationBatchler(9, rows8={"x": 45}).process(mixed)])
    assert torch.equal(out.double(), exact_values(torch.cat([data[0]["x"], data[1]["x"]])))


def test_buffer_refusals(pkg):
    go = lambda *chunks: list(pkg.ActivationBatchler(4, rows8={"x": 45}).process([{"x": c} for c in chunks]))  # noqa: E731
    for bad in (rows(5, 44, 0), torch.zeros(5, 45, dtype=torch.int32), rows(5, 45, 0)[:, None], torch.zeros(5, 64, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            go(bad)
        with pytest.raises((ValueError, AssertionError)):
            go(rows(5, 45, 0), bad)
    with pytest.raises(ValueError):
        go(rows(5, 45, 0), torch.zeros(5, 1, dtype=torch.uint8))


def test_loader_refuses_files_that_disagree(pkg, tmp_path):
    from safetensors.torch import load_file, save_file

    w = lambda **kw: pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path), hook_points=["h0"], **kw))  # noqa: E731
    w(row_format="rows8").process(samples(2, 4, 40))
    second = tmp_path / "h0" / "chunk-00000001.safetensors"
    good = load_file(str(second))
    load = lambda: list(pkg.CachedActivationLoader({"h0": tmp_path / "h0"}).process())  # noqa: E731
    assert len(load()) == 2
    for change in ({"activation_width": torch.tensor([41, 0])}, {"activation_width": torch.tensor([80, 0])},
                   {"activation_width": torch.tensor([40, 9])}, {"activation": torch.zeros(1, 4, 40)},
                   {"activation": torch.zeros(1, 4, 48, dtype=torch.uint8), "activation_width": torch.tensor([20, 0])}):
        save_file(good | change, str(second))
        with pytest.raises(ValueError, match="cached activation"):
            load()
    save_file({k: v for k, v in good.items() if k != "activation_width"}, str(second))
    with pytest.raises(ValueError, match="float rows after"):
        load()
    with pytest.raises(ValueError):
        w(row_format="rows8").process([{"h0": torch.zeros(1, 4, 8, dtype=torch.float64), "tokens": torch.zeros(1, 4)}])
    with pytest.raises(ValueError):
        w(row_format="int4")


def write_chunks(pkg, path, parts):
    """One chunk of two samples per part (d, dtype, row format): -> the float rows that each is to come out as."""
    want = []
    for i, (d, dtype, form) in enumerate(parts):
        part = list(samples(2, 4, d, dtype))
        part[0]["h0"][0, 0, 0] = 1e5 if dtype != torch.float16 else 6e4        # past fp16's largest where the type holds it
        pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(path), hook_points=["h0"], n_samples_per_chunk=2, row_format=form)
                             ).process(part, start_shard=i)
        x = torch.cat([s["h0"] for s in part])
        want.append(exact_values(x.reshape(-1, d)).view(x.shape).to(dtype) if form == "rows8" else x)
    return want


def read_ahead(loader):
    """All chunks as a reader thread far ahead of its consumer leaves them: every one read before the first is handed over."""
    chunks = {hp: loader._get_sorted_chunks(hp) for hp in loader.cache_dirs}
    widths = {}
    held = [loader._read_chunk_index(i, chunks, widths) for i in range(len(chunks["h0"]))]
    return [loader._floats(c) for c in held]


MIXED = [[(40, torch.bfloat16, "rows8"), (40, torch.float16, "rows8"), (40, torch.float32, "rows8")],
         [(40, torch.float32, "float"), (40, torch.bfloat16, "rows8")],
         [(24, torch.bfloat16, "float"), (40, torch.float32, "rows8"), (40, torch.bfloat16, "rows8")]]


@pytest.mark.parametrize("parts", MIXED)
def test_chunks_are_read_back_as_they_were_written(pkg, tmp_path, parts):
    """The type and form of a chunk do not depend on how far ahead of it the reader is, nor on an earlier pass."""
    want = write_chunks(pkg, tmp_path, parts)
    loader = pkg.CachedActivationLoader({"h0": tmp_path / "h0"})
    for got in (list(loader.process()), read_ahead(loader), list(loader.process())):
        assert len(got) == len(parts)
        for a, b in zip(got, want):
            assert set(a) == {"tokens", "mask", "attention_mask", "meta", "h0"}
            assert a["h0"].dtype == b.dtype and torch.equal(a["h0"], b)
    for a, b in zip(pkg.CachedActivationLoader({"h0": tmp_path / "h0"}, dtype=torch.float32).process(), want):
        assert a["h0"].dtype == torch.float32 and torch.equal(a["h0"], b.float())


@pytest.mark.parametrize("first,second", [("float", "rows8"), ("rows8", "float")])
def test_records_that_are_kept_do_not_mix_with_floats(pkg, tmp_path, first, second):
    write_chunks(pkg, tmp_path, [(40, torch.float32, first), (40, torch.float32, second)])
    loader = pkg.CachedActivationLoader({"h0": tmp_path / "h0"}, keep_rows8=True)
    for _ in range(2):      # every pass starts anew
        it = loader.process()
        assert next(it)["h0"].dtype == (torch.uint8 if first == "rows8" else torch.float32)
        with pytest.raises(ValueError, match="float rows"):
            next(it)


def test_widths_follow_the_files(pkg, tmp_path):
    """A directory that is written anew in another form or width is read as it is."""
    loader = pkg.CachedActivationLoader({"h0": tmp_path / "h0"}, keep_rows8=True)
    for d, form in ((40, "rows8"), (70, "rows8"), (70, "float"), (40, "rows8")):
        write_chunks(pkg, tmp_path, [(d, torch.float32, form)])
        (got,) = loader.process()
        assert loader.rows8_widths == ({"h0": d} if form == "rows8" else {})
        assert got["h0"].shape[-1] == (pkg.ops.rows8_pitch(d) if form == "rows8" else d)
