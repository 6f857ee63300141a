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


def test_rows8_holds_whole_records(pkg):
    R = pkg.Rows8
    ok = R(torch.zeros(3, 80, dtype=torch.uint8), 40)
    assert ok.shape == (3, 40) and len(ok) == 3 and ok.device.type == "cpu"
    for data, d in [(torch.zeros(3, 80), 40), (torch.zeros(3, 96, dtype=torch.uint8), 40), (torch.zeros(80, dtype=torch.uint8), 40),
                    (torch.zeros(3, 48, dtype=torch.uint8), 40), (torch.zeros(3, 0, dtype=torch.uint8), 0)]:
        with pytest.raises(ValueError):
            R(data, d)


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
    assert ot(s=0) == -1 and ot(s=2) == -1 and ot(s=3, part=P) == -1 and ot(n=1 << 22) == -2 and ot(m=1 << 29) == -2
    need = lib.sae_rows8_grad_rows_workspace_bytes(100, 40)
    assert need >= 100 * 4 and lib.sae_rows8_grad_rows_workspace_bytes(0, 40) == 0
    rows = lambda r=P, out=P, F=4, d=40, n=100, ws=P, b=need: lib.sae_rows8_grad_rows(P, P, P, P, r, out, None, F, d, n, ws, b, None)  # noqa: E731
    assert rows(r=None) == -1 and rows(out=None) == -1 and rows(F=0) == -1 and rows(d=0) == -1 and rows(n=0) == -1
    assert rows(r=P + 8) == -1 and rows(ws=None) == -4 and rows(b=need - 1) == -4 and rows(d=1 << 30) == -2 and rows(n=(1 << 31) - 1) == -2
    assert lib.sae_sparse_grad_rows(P, P, P, P, P, 2, P, None, 4, 40, None) == -1      # records have their own entry point
