"""Rows held in 8 bits on the GPU: writing, reading, transposing, dense and sparse weight gradients, the Adam and norm passes
over them, against plain implementations in 64 bits."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


# ---- the format, from its definition, in 64 bits -------------------------------------------------------------

def pitch_of(d):
    nb = -(-d // 32)
    return -(-(33 * nb) // 16) * 16


def record_of(x):
    """(codes int64 [n, 32 nb], fields int64 [n, nb]) of a float array, block by block."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    nb = -(-d // 32)
    full = np.zeros((n, 32 * nb))
    full[:, :d] = x
    blocks = full.reshape(n, nb, 32)
    codes, fields = np.zeros((n, nb, 32), dtype=np.int64), np.zeros((n, nb), dtype=np.int64)
    top = np.abs(blocks).max(2)
    bad = ~np.isfinite(blocks).all(2)
    fields[bad] = 255
    live = ~bad & (top > 0)
    if live.any():
        t = top[live]
        k = np.maximum(np.floor(np.log2(t)).astype(np.int64) - 6, -126)
        k = np.where((np.rint(np.ldexp(t, -k)) > 127) & (k < 121), k + 1, k)
        fields[live] = k + 127
        codes[live] = np.clip(np.rint(np.ldexp(blocks[live], -k[:, None])), -127, 127).astype(np.int64)
    return codes.reshape(n, 32 * nb), fields


def values_of(codes, fields, d):
    step = np.where(fields == 0, 0.0, np.where(fields == 255, np.nan, np.ldexp(1.0, (fields - 127).astype(int))))
    return (codes.reshape(*fields.shape, 32) * step[:, :, None]).reshape(codes.shape[0], -1)[:, :d]


def unpack(rows8):
    data = rows8.data.cpu().numpy()
    nb = -(-rows8.d // 32)
    return data[:, : 32 * nb].view(np.int8).astype(np.int64), data[:, 32 * nb : 33 * nb].astype(np.int64), data[:, 33 * nb :]


def activations(n, d, seed, dtype=torch.float32, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(n, d, generator=g, device=dev) * torch.exp(torch.randn(n, 1, generator=g, device=dev))
    x[:, d // 2] *= 50.0
    return x.to(dtype)


def doubles(t):
    return t.detach().double().cpu().numpy()


# ---- writing -----------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (3, 31), (2, 32), (5, 33), (1, 64), (7, 100), (64, 768), (33, 1037), (4, 4096), (2, 8193), (300, 48)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", SHAPES)
def test_records_are_the_definitions(pkg, dev, n, d, dtype):
    x = activations(n, d, 1, dtype)
    q = pkg.ops.quantize_rows(x)
    assert q.shape == (n, d) and tuple(q.data.shape) == (n, pitch_of(d)) == (n, pkg._lib.load().sae_rows8_pitch(d))
    codes, fields, tail = unpack(q)
    want_codes, want_fields = record_of(doubles(x))
    np.testing.assert_array_equal(fields, want_fields)
    np.testing.assert_array_equal(codes, want_codes)
    assert not tail.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gap,first", [(0, 0), (1, 0), (37, 0), (8, 1), (5, 3)])
def test_rows_of_a_wider_tensor(pkg, dev, gap, first, dtype):
    """Rows lie any distance apart and start anywhere; a row may be repeated by a stride of 0."""
    wide = activations(19, 130 + gap + first, 2, dtype)
    x = wide[:, first : first + 130]
    assert torch.equal(pkg.ops.quantize_rows(x).data, pkg.ops.quantize_rows(x.contiguous()).data)
    one = x[:1].expand(6, 130)
    assert torch.equal(pkg.ops.quantize_rows(one).data, pkg.ops.quantize_rows(x[:1]).data.expand(6, -1))


def test_extremes(pkg, dev):
    """Borders of the step, denormals, the largest float, infinities and NaN, signed zeros; blocks do not touch each other."""
    f32 = np.float32
    top = float(np.finfo(f32).max)
    edge = [127.5 / 64, np.nextafter(f32(127.5 / 64), f32(0)), 1.0, np.nextafter(f32(1), f32(0)), 2.0**-120, 2.0**-121,
            2.0**-126, 2.0**-127, 2.0**-128, 1e-44, top, top / 2, 127.4 * 2.0**121, 127.5 * 2.0**121, 0.0, -0.0,
            float("inf"), float("-inf"), float("nan")]
    rows = []
    for e in edge:
        r = np.zeros(96, dtype=f32)
        r[5], r[6], r[7] = e, -e / 3, e / 255
        r[32:64] = np.linspace(-1, 1, 32)
        r[64] = -e
        rows.append(r)
    x = torch.from_numpy(np.stack(rows)).to(dev)
    q = pkg.ops.quantize_rows(x)
    codes, fields, _ = unpack(q)
    want_codes, want_fields = record_of(doubles(x))
    np.testing.assert_array_equal(fields, want_fields)
    np.testing.assert_array_equal(codes, want_codes)
    back = pkg.ops.restore_rows(q, torch.float32)
    np.testing.assert_array_equal(doubles(back), values_of(codes, fields, 96))
    finite = torch.isfinite(x).all(1)
    assert torch.isfinite(back[finite]).all() and back[~finite, :32].isnan().all() and torch.isfinite(back[~finite, 32:64]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_error_is_half_a_step_and_rewriting_changes_nothing(pkg, dev, dtype):
    x = activations(200, 515, 3, dtype)
    q = pkg.ops.quantize_rows(x)
    _, fields, _ = unpack(q)
    step = np.ldexp(1.0, fields - 127).repeat(32, 1)[:, :515]
    back = pkg.ops.restore_rows(q, torch.float32)
    assert (np.abs(doubles(back) - doubles(x)) <= step / 2).all()
    b16 = pkg.ops.restore_rows(q)
    assert b16.dtype == torch.bfloat16 and torch.equal(b16.float(), back)          # exact in bf16
    again = pkg.ops.quantize_rows(b16)
    assert torch.equal(pkg.ops.restore_rows(again, torch.float32), back)


@pytest.mark.parametrize("n,d", [(1, 1), (9, 77), (64, 768), (5, 4100)])
def test_the_operand_copy_is_the_rounded_source(pkg, dev, n, d):
    x = activations(n, d + 3, 4)[:, :d]
    q, copy = pkg.ops.quantize_rows(x, bf16_copy=True)
    assert torch.equal(copy, x.to(torch.bfloat16)) and torch.equal(q.data, pkg.ops.quantize_rows(x).data)
    y = x.to(torch.bfloat16).contiguous()
    q2, copy2 = pkg.ops.quantize_rows(y, bf16_copy=True)
    assert copy2 is y and torch.equal(q2.data, pkg.ops.quantize_rows(y).data)
    z = activations(n, d + 3, 4, torch.bfloat16)[:, :d]
    q3, copy3 = pkg.ops.quantize_rows(z, bf16_copy=True)
    assert torch.equal(copy3, z) and copy3.is_contiguous() and torch.equal(q3.data, pkg.ops.quantize_rows(z).data)


def test_writing_into_a_buffer_leaves_the_other_rows(pkg, dev):
    slab = torch.full((20, pitch_of(100)), 7, dtype=torch.uint8, device=dev)
    x = activations(6, 100, 5)
    pkg.ops.quantize_rows(x, out=slab[9:15])
    assert torch.equal(slab[9:15], pkg.ops.quantize_rows(x).data) and (slab[:9] == 7).all() and (slab[15:] == 7).all()


# ---- reading -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.37, -3.0])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 31), (40, 768), (17, 1037), (3, 4096), (2, 8193)])
def test_gather(pkg, dev, n, d, scale, out_dtype):
    q = pkg.ops.quantize_rows(activations(50, d, 6))
    codes, fields, _ = unpack(q)
    values = values_of(codes, fields, d)
    idx = torch.randint(0, 50, (n,), device=dev)            # the same row several times, in any order
    got = pkg.ops.gather_rows(q, idx, out_dtype, scale)
    want = torch.from_numpy(values[idx.cpu().numpy()]).float() * torch.tensor(scale, dtype=torch.float32)   # one fp32 rounding
    assert torch.equal(got.cpu(), want.to(out_dtype))
    out = torch.empty_like(got)
    assert pkg.ops.gather_rows(q, idx, out_dtype, scale, out=out) is out and torch.equal(out, got)


def test_a_row_outside_the_buffer_reads_as_nan(pkg, dev):
    q = pkg.ops.quantize_rows(activations(8, 70, 7))
    part = pkg.ops.Rows8(q.data[2:6], 70)                   # its neighbours are there, and are not read
    idx = torch.tensor([0, -1, 3, 4, 2**40, -(2**40)], device=dev)
    got = pkg.ops.gather_rows(part, idx, torch.float32)
    whole = pkg.ops.restore_rows(q, torch.float32)
    assert torch.equal(got[0], whole[2]) and torch.equal(got[2], whole[5])
    assert got[[1, 3, 4, 5]].isnan().all()


def test_offsets_past_32_bits(pkg, dev):
    """A buffer of 5 GB whose last rows lie behind 2^32 bytes."""
    d, n = 4096, 1_200_000
    data = torch.empty(n, pitch_of(d), dtype=torch.uint8, device=dev)
    x = activations(8, d, 8)
    pkg.ops.quantize_rows(x, out=data[n - 8 :])
    pkg.ops.quantize_rows(x.flip(0), out=data[:8])
    idx = torch.tensor([n - 1, 0, n - 8, 7], device=dev)
    want = pkg.ops.restore_rows(pkg.ops.quantize_rows(x), torch.float32)
    got = pkg.ops.gather_rows(pkg.ops.Rows8(data, d), idx, torch.float32)
    assert torch.equal(got, want[[7, 7, 0, 0]])


def test_more_pieces_than_one_launch_counts(pkg, dev):
    """2^27 rows of 32 fp32 values are 2^30 pieces, the most of one launch: rows behind them go through a second one."""
    ops = pkg.ops
    n, d = (1 << 27) + 5, 32
    base = torch.randn(n + d - 1, generator=torch.Generator(device=dev).manual_seed(6), device=dev)
    x = base.as_strided((n, d), (1, 1))                  # row i: the 32 values from the i-th on
    q = ops.quantize_rows(x)
    out = ops.restore_rows(q, torch.float32)
    for at in (0, 12345, (1 << 27) - 3, n - 6):
        some = slice(at, at + 6)
        want = ops.quantize_rows(x[some].contiguous())
        assert torch.equal(q.data[some], want.data)
        assert torch.equal(out[some], ops.restore_rows(want, torch.float32))
    del out, x, base
    idx = torch.arange(n - 1, -1, -1, device=dev)
    got = ops.gather_rows(q, idx, torch.float32)
    for at in (0, 777, (1 << 27) - 3, n - 6):
        some = slice(at, at + 6)
        assert torch.equal(got[some], ops.gather_rows(q, idx[some].contiguous(), torch.float32))


# ---- dense weight gradients ------------------------------------------------------------------------------------

def bound(left, right, terms):
    """|fp32 sum - exact| <= 2 terms 2^-24 sum |l| |r|: each of the `terms` additions rounds (or, inside a matrix
    instruction, truncates) once."""
    return 2.0 * terms * 2.0**-24 * (np.abs(left).T @ np.abs(right)) + 1e-40


@pytest.mark.parametrize("T,m,n", [(1, 1, 1), (1, 40, 33), (63, 8, 64), (64, 64, 64), (65, 130, 37), (200, 520, 96), (512, 256, 768),
                                   (1000, 1003, 521)])
@pytest.mark.parametrize("left_kind", ["bf16", "f32", "rows8"])
def test_gemm_over_tokens(pkg, dev, T, m, n, left_kind):
    ops = pkg.ops
    left = activations(T, m, 9, torch.float32) * 1e-3
    right = ops.quantize_rows(activations(T, n, 10))
    r = doubles(ops.restore_rows(right, torch.float32))
    if left_kind == "rows8":
        left = ops.quantize_rows(left)
        lv = doubles(ops.restore_rows(left, torch.float32))
    else:
        left = left.to(torch.bfloat16) if left_kind == "bf16" else left
        lv = doubles(left)
    got = doubles(ops.gemm_over_tokens(left, right))
    assert got.shape == (m, n)
    assert (np.abs(got - lv.T @ r) <= bound(lv, r, T)).all()
    swapped = doubles(ops.gemm_over_tokens(right, left))
    assert (np.abs(swapped - r.T @ lv) <= bound(r, lv, T)).all()
    if left_kind != "f32":
        low = doubles(ops.gemm_over_tokens(left, right, torch.bfloat16))
        want = lv.T @ r
        assert (np.abs(low - want) <= bound(lv, r, T) + 2.0**-8 * np.abs(want) + 1e-38).all()


@pytest.mark.parametrize("T,m,n", [(2049, 4100, 2055), (2112, 4096, 2048), (2500, 2056, 3600)])
@pytest.mark.parametrize("left_kind", ["bf16", "rows8"])
def test_large_products(pkg, dev, T, m, n, left_kind):
    """Past the size that the 64 x 64 tiles take: tokens and widths that the GEMM kernel's slabs divide, or do not."""
    ops = pkg.ops
    assert 2.0 * (T + 1000) * m * n > ops.OVER_TOKENS_FLOP
    left, right = activations(T, m, 9, torch.bfloat16), ops.quantize_rows(activations(T, n, 10))
    left = ops.quantize_rows(left) if left_kind == "rows8" else left
    lv = (ops.restore_rows(left, torch.float32) if left_kind == "rows8" else left).double()
    r = ops.restore_rows(right, torch.float32).double()
    limit = 2.0 * T * 2.0**-24 * (lv.abs().t() @ r.abs()) + 1e-40
    assert ((ops.gemm_over_tokens(left, right).double() - lv.t() @ r).abs() <= limit).all()
    assert ((ops.gemm_over_tokens(right, left).double() - r.t() @ lv).abs() <= limit.t()).all()


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,m,n", [(8192, 2048, 1536), (8192, 1111, 2500), (8130, 2056, 1532)])
def test_large_products_of_few_tiles(pkg, dev, T, m, n, out_dtype):
    """Few 256 x 256 tiles over many tokens: slices of the tokens, joined in order."""
    ops = pkg.ops
    assert 2.0 * (T + 1000) * m * n > ops.OVER_TOKENS_FLOP and ops.gemm_split_k(m, -(-T // 64) * 64, n) > 1
    left, right = activations(T, m, 11, torch.bfloat16), ops.quantize_rows(activations(T, n, 12))
    r = ops.restore_rows(right, torch.float32).double()
    want, size = left.double().t() @ r, left.double().abs().t() @ r.abs()
    got = ops.gemm_over_tokens(left, right, out_dtype)
    assert got.dtype == out_dtype and torch.equal(got, ops.gemm_over_tokens(left, right, out_dtype))
    low = 2.0**-8 * want.abs() if out_dtype == torch.bfloat16 else 0.0
    assert ((got.double() - want).abs() <= 2.0 * T * 2.0**-24 * size + low + 1e-38).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.gemm_over_tokens(left, right, out_dtype)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, got) and torch.equal(ops.gemm_over_tokens(left, right, out_dtype), got)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("slices", [1, 2, 3, 7])
def test_slices_of_the_tokens(pkg, dev, slices, wide):
    """Any number of slices of whole slabs, the last one short, adds up to the same product."""
    ops, lib = pkg.ops, pkg._lib.load()
    T, m, n = 450, 70, 45
    left = activations(T, m, 11, torch.float32 if wide else torch.bfloat16)
    right = ops.quantize_rows(activations(T, n, 12))
    out, part = torch.full((m, n), float("nan"), device=dev), torch.full((slices, m, n), float("nan"), device=dev)
    pkg._lib.check(lib.sae_gemm_over_tokens(left.data_ptr(), 0 if wide else 1, right.data.data_ptr(), 2, T, m, n, out.data_ptr(), 0, slices,
                                            part.data_ptr(), torch.cuda.current_stream().cuda_stream))
    lv, r = doubles(left), doubles(ops.restore_rows(right, torch.float32))
    assert (np.abs(doubles(out) - lv.T @ r) <= bound(lv, r, T)).all()


def test_gemm_over_tokens_of_float_operands(pkg, dev):
    """Any two operand types; rows that 8 bits hold exactly give the product of the float rows, bit for bit."""
    ops = pkg.ops
    left, right = ops.quantize_rows(activations(300, 76, 11)), ops.quantize_rows(activations(300, 100, 12))
    forms = lambda q: (q, ops.restore_rows(q), ops.restore_rows(q, torch.float32))  # noqa: E731
    low = [ops.gemm_over_tokens(a, b) for a in forms(left)[:2] for b in forms(right)[:2]]
    wide = [ops.gemm_over_tokens(a, b) for a in forms(left) for b in forms(right) if torch.float32 in (getattr(a, "dtype", 0), getattr(b, "dtype", 0))]
    assert len(low) == 4 and len(wide) == 5
    for group in (low, wide):
        for g in group[1:]:
            assert torch.equal(g, group[0])


def test_the_two_tilings_agree(pkg, dev, monkeypatch):
    ops = pkg.ops
    left, right = activations(256, 160, 13, torch.bfloat16), ops.quantize_rows(activations(256, 96, 14))
    small = doubles(ops.gemm_over_tokens(left, right))
    monkeypatch.setattr(ops, "OVER_TOKENS_FLOP", 0.0)
    large = ops.gemm_over_tokens(left, right)
    assert torch.equal(large, ops.gemm(left, ops.restore_rows(right), torch.float32, True, True))
    assert (np.abs(small - doubles(large)) <= bound(doubles(left), doubles(ops.restore_rows(right, torch.float32)), 256)).all()


def test_out_of_an_odd_width_starts_anywhere(pkg, dev):
    ops = pkg.ops
    q = ops.quantize_rows(activations(50, 37, 26))
    code = sparse_code(ops, 50, 9, 3, 27, dev)
    fi = ops.build_feature_index(code)
    frame = torch.full((11, 37), 7.0, device=dev)
    rows, _ = ops.sparse_grad_rows(fi, code.val, q, 9, out=frame[1:10])
    assert torch.equal(rows, ops.sparse_grad_rows(fi, code.val, q, 9)[0]) and (frame[0] == 7).all() and (frame[10] == 7).all()


@pytest.mark.parametrize("left_kind", ["bf16", "f32", "rows8"])
@pytest.mark.parametrize("T,m,n", [(700, 1, 1), (700, 3, 2), (257, 5, 31), (129, 7, 70), (640, 2, 130), (66, 1, 9)])
def test_products_of_few_columns(pkg, dev, T, m, n, left_kind):
    """Rows shorter than one load: what it reads behind a row enters no sum."""
    ops = pkg.ops
    left = activations(T, m, 81, torch.float32 if left_kind == "f32" else torch.bfloat16)
    left_q = ops.quantize_rows(left) if left_kind == "rows8" else left
    right = ops.quantize_rows(activations(T, n, 82))
    values = doubles(ops.restore_rows(left_q, torch.float32)) if left_kind == "rows8" else doubles(left)
    r = doubles(ops.restore_rows(right, torch.float32))
    got = doubles(ops.gemm_over_tokens(left_q, right))
    # bf16 and 8-bit operands: exact products; fp32: products rounded once; sums of T terms
    assert (np.abs(got - values.T @ r) <= 2 * (T + 1) * 2.0**-24 * (np.abs(values).T @ np.abs(r)) + 1e-30).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_what_is_not_finite_stays_in_its_row_and_column(pkg, dev, kind):
    """A NaN in the first column of a row lies right behind the row before it, and one in the last token in the last slab."""
    ops = pkg.ops
    T, m, n = 203, 131, 69
    left, right = activations(T, m, 83, kind), activations(T, n, 84)
    want = ops.gemm_over_tokens(left, ops.quantize_rows(right))
    left[90, 0] = float("nan")
    left[T - 1, m - 1] = float("inf")
    got = ops.gemm_over_tokens(left, ops.quantize_rows(right))
    assert not torch.isfinite(got[0]).any() and not torch.isfinite(got[m - 1]).any()
    assert torch.equal(got[1:-1], want[1:-1])
    held_nan = right.clone()
    held_nan[5, 3] = float("nan")                        # its block of 32 values
    got = ops.gemm_over_tokens(activations(T, m, 83, kind), ops.quantize_rows(held_nan))
    assert torch.isnan(got[:, :32]).all() and torch.equal(got[:, 32:], want[:, 32:])


def whole(shape, seed, dev, top=2):
    """Whole numbers up to `top`: every product and sum of few of them is exact in any order, in bf16 products too."""
    return torch.randint(-top, top + 1, shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).float()


@pytest.mark.parametrize("T,m,n", [(64, 4300000, 4), (65, 3, 4300001), (1, 4194241, 1), (2, 1, 4194241)])
@pytest.mark.parametrize("kind", ["bf16", "f32", "rows8"])
def test_products_of_very_wide_operands(pkg, dev, T, m, n, kind):
    ops = pkg.ops
    left, right = whole((T, m), 1, dev), whole((T, n), 2, dev)
    want = left.t() @ right
    make = {"bf16": lambda x: x.bfloat16(), "f32": lambda x: x, "rows8": ops.quantize_rows}[kind]
    got = ops.gemm_over_tokens(make(left), ops.quantize_rows(right))
    assert got.dtype == torch.float32 and got.is_contiguous() and torch.equal(got, want)
    got = ops.gemm_over_tokens(ops.quantize_rows(left), make(right), torch.float32 if kind == "f32" else torch.bfloat16)
    assert got.is_contiguous() and torch.equal(got.float(), want.to(got.dtype).float())


@pytest.mark.parametrize("kind", ["bf16", "rows8"])
def test_products_over_very_many_tokens(pkg, dev, kind):
    """More tokens than one grid axis of 128-token tiles counts; sums of ones, exact in fp32 in any order."""
    ops = pkg.ops
    T, m, n = 65535 * 128 + 77, 72, 66
    left, right = whole((T, m), 3, dev, 1).bfloat16(), whole((T, n), 4, dev, 1)
    q, l8 = ops.quantize_rows(right), ops.quantize_rows(left)
    assert 2.0 * T * m * n > ops.OVER_TOKENS_FLOP
    want = torch.zeros(m, n, dtype=torch.float64, device=dev)
    for t in range(0, T, 1 << 20):
        want += left[t : t + (1 << 20)].double().t() @ right[t : t + (1 << 20)].double()
    got = ops.gemm_over_tokens(left if kind == "bf16" else l8, q)
    assert torch.equal(got.double(), want)


def test_no_tokens(pkg, dev):
    ops = pkg.ops
    q = ops.quantize_rows(torch.empty(0, 40, device=dev))
    assert q.shape == (0, 40) and ops.restore_rows(q).shape == (0, 40)
    assert ops.gather_rows(q, torch.empty(0, dtype=torch.int64, device=dev)).shape == (0, 40)
    out = ops.gemm_over_tokens(torch.empty(0, 24, dtype=torch.bfloat16, device=dev), q)
    assert out.shape == (24, 40) and not out.any()


# ---- sparse weight gradients --------------------------------------------------------------------------------------

def sparse_code(ops, T, F, k, seed, dev, heavy=False):
    """A code whose first feature is kept by every token when `heavy`; features behind F - 3 are never kept."""
    g = torch.Generator(device=dev).manual_seed(seed)
    score = torch.rand(T, F, generator=g, device=dev)
    if F > 3:
        score[:, F - 3 :] = -1.0
    if heavy:
        score[:, 0] = 2.0
    idx = score.topk(k, 1).indices.sort(1).values.to(torch.int32)
    nnz = torch.randint(0, k + 1, (T,), generator=g, device=dev, dtype=torch.int32)     # some tokens keep nothing
    if heavy:
        nnz.clamp_(min=1)
    slot = torch.arange(k, device=dev)[None, :]
    val = torch.randn(T, k, generator=g, device=dev)
    val[slot >= nnz[:, None]] = 0.0
    idx[slot >= nnz[:, None]] = 0
    return ops.SparseCode(idx.reshape(-1).contiguous(), val.reshape(-1).contiguous(), torch.arange(T, device=dev) * k, nnz, T, F)


CODES = [(96, 30, 9, 40), (120, 30, 9, 40), (90, 3000, 5, 700), (1024, 130, 4, 40), (1025, 130, 4, 40), (900, 512, 8, 517), (333, 41, 3, 1030), (1, 5, 1, 40), (7, 30, 4, 33), (64, 100, 8, 768), (300, 17, 5, 1037), (513, 64, 12, 520), (1500, 12, 3, 2052), (40, 9, 2, 4100),
         (33, 50, 6, 1), (128, 5, 1, 64), (2000, 400, 16, 260), (640, 8, 5, 36), (4096, 3, 1, 300),
         (4100, 60, 32, 1500), (9000, 300, 48, 516)]


@pytest.mark.parametrize("heavy", [False, True])
@pytest.mark.parametrize("T,F,k,d", CODES)
def test_gradient_rows(pkg, dev, T, F, k, d, heavy):
    ops = pkg.ops
    q = ops.quantize_rows(activations(T, d, 13))
    code = sparse_code(ops, T, F, k, 14, dev, heavy)
    fi = ops.build_feature_index(code)
    out, bias = ops.sparse_grad_rows(fi, code.val, q, F, want_bias=True)
    dense = doubles(code.to_dense())
    values = doubles(ops.restore_rows(q, torch.float32))
    per_feature = (dense != 0).sum(0)[:, None] + 1
    assert (np.abs(doubles(out) - dense.T @ values) <= 2.0**-23 * per_feature * (np.abs(dense).T @ np.abs(values)) + 1e-40).all()
    assert (np.abs(doubles(bias) - dense.sum(0)) <= 2.0**-23 * per_feature[:, 0] * np.abs(dense).sum(0) + 1e-40).all()
    assert not out[(dense == 0).all(0)].any()               # features that no token kept
    if d % 4 == 0:                                          # the same rows held in floats: the same bits, but for features whose
        ptr = fi.feat_ptr.long()                            # slots cross a multiple of 32, which may be summed in pieces
        whole = (ptr[:-1] // 32 == (ptr[1:] - 1).clamp_min(0) // 32) | (ptr[:-1] == ptr[1:])
        floats = ops.restore_rows(q)
        want, _ = ops.sparse_grad_rows(fi, code.val, floats, F)
        assert torch.equal(out[whole], want[whole])
        wide, _ = ops.sparse_grad_rows(fi, code.val, floats.float(), F)
        assert torch.equal(out[whole], wide[whole])
    again, _ = ops.sparse_grad_rows(fi, code.val, q, F)
    assert torch.equal(out, again)                          # the order of every sum is fixed


def test_gradient_rows_of_the_longest_index(pkg, dev):
    """131072 tokens, the most a feature index takes, one feature kept by all of them."""
    ops = pkg.ops
    T, F, k, d = 131072, 200, 3, 70
    q = ops.quantize_rows(activations(T, d, 15))
    code = sparse_code(ops, T, F, k, 16, dev, True)
    fi = ops.build_feature_index(code)
    out, bias = ops.sparse_grad_rows(fi, code.val, q, F, want_bias=True)
    dense, values = code.to_dense().double(), ops.restore_rows(q, torch.float32).double()
    kept = (dense != 0).sum(0)
    assert kept.max() == T
    size = dense.abs().t() @ values.abs()
    assert ((out.double() - dense.t() @ values).abs() <= 2.0**-23 * (kept[:, None] + 1) * size + 1e-40).all()
    assert ((bias.double() - dense.sum(0)).abs() <= 2.0**-23 * (kept + 1) * dense.abs().sum(0) + 1e-40).all()
    again, _ = ops.sparse_grad_rows(fi, code.val, q, F)
    assert torch.equal(out, again)


@pytest.mark.parametrize("lowp", [False, True])
@pytest.mark.parametrize("d", [64, 516, 768, 1024, 2048, 4096])
def test_adam_and_norm_over_8_bit_rows(pkg, dev, d, lowp):
    """The passes that rebuild a gradient row on the way read 8-bit rows as they read the bf16 rows they stand for: same bits."""
    ops = pkg.ops
    T, F, k = 150, 40, 6
    q = ops.quantize_rows(activations(T, d, 15))
    floats = ops.restore_rows(q)
    code = sparse_code(ops, T, F, k, 16, dev, True)
    fi = ops.build_feature_index(code)
    dt = torch.bfloat16 if lowp else torch.float32
    results = []
    for dense in (q, floats):
        g = torch.Generator(device=dev).manual_seed(17)
        p = torch.randn(F, d, generator=g, device=dev).to(dt)
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        bias, norm = torch.empty(F, device=dev), torch.empty(F, device=dev)
        acc = torch.zeros(2, dtype=torch.float64, device=dev)
        ops.adam_step_sparse_rows(fi, code.val, dense, p, m, v, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=3, bias_grad_out=bias,
                                  row_norm_out=norm, grad_sq_nnz_acc=acc)
        sums, bias2 = torch.zeros(2, dtype=torch.float64, device=dev), torch.empty(F, device=dev)
        ops.sparse_rows_grad_sq_nnz(fi, code.val, dense, sums, bias_grad_out=bias2)
        results.append((p, m, v, bias, norm, acc, sums, bias2))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lowp", [False, True])
@pytest.mark.parametrize("T,d", [(517, 64), (700, 768), (1030, 1028), (603, 2052)])
def test_adam_and_norm_over_long_segments_of_8_bit_rows(pkg, dev, T, d, lowp):
    """Features that nearly all tokens keep: segments of more than two chunks of looked-up slots (192 or 256 each), and ragged ends.
    The same bits as over the bf16 rows; the gradient's square sum and the bias gradient against 64-bit sums."""
    ops = pkg.ops
    F, k = 24, 6
    q = ops.quantize_rows(activations(T, d, 31))
    floats = ops.restore_rows(q)
    code = sparse_code(ops, T, F, k, 32, dev, True)
    fi = ops.build_feature_index(code)
    longest = int((fi.feat_ptr[1:] - fi.feat_ptr[:-1]).max())
    assert longest > 512 and longest % 8
    dt = torch.bfloat16 if lowp else torch.float32
    results = []
    for dense in (q, floats):
        g = torch.Generator(device=dev).manual_seed(33)
        p = torch.randn(F, d, generator=g, device=dev).to(dt)
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        bias, norm = torch.empty(F, device=dev), torch.empty(F, device=dev)
        acc = torch.zeros(2, dtype=torch.float64, device=dev)
        ops.adam_step_sparse_rows(fi, code.val, dense, p, m, v, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=3, bias_grad_out=bias,
                                  row_norm_out=norm, grad_sq_nnz_acc=acc)
        sums, bias2 = torch.zeros(2, dtype=torch.float64, device=dev), torch.empty(F, device=dev)
        ops.sparse_rows_grad_sq_nnz(fi, code.val, dense, sums, bias_grad_out=bias2)
        results.append((p, m, v, bias, norm, acc, sums, bias2))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    coef = torch.zeros(F, T, dtype=torch.float64, device=dev)
    tok = fi.slot_tok.long()
    coef.index_put_((code.idx.long(), tok), code.val.double(), accumulate=True)
    grad, size = coef @ floats.double(), coef.abs() @ floats.double().abs()
    _, _, _, bias, _, acc, sums, bias2 = results[0]
    # an entry: one rounding of each of at most `longest` additions; where the state is bf16 the Adam pass rounds the sum to bf16
    off = 1.01 * longest * 2.0**-24 * size
    low = off + (2.0**-8 * (grad.abs() + off) if lowp else 0.0)
    for total, e in ((acc[0], low), (sums[0], off)):       # squares added by fours in fp32, those in 64 bits
        assert (total - grad.square().sum()).abs() <= (2 * grad.abs() * e + e * e).sum() + 4 * 2.0**-24 * (grad.abs() + e).square().sum()
    b_sum, b_off = coef.sum(1), 1.01 * longest * 2.0**-24 * coef.abs().sum(1)
    assert ((bias.double() - b_sum).abs() <= b_off).all() and ((bias2.double() - b_sum).abs() <= b_off).all()


def test_blocks_that_are_not_finite_stay_in_their_rows(pkg, dev):
    ops = pkg.ops
    x = activations(6, 96, 18)
    x[2, 40] = float("inf")
    x[4, 3] = float("nan")
    q = ops.quantize_rows(x)
    code = ops.SparseCode(torch.arange(6, dtype=torch.int32, device=dev), torch.ones(6, device=dev), torch.arange(6, device=dev),
                          torch.ones(6, dtype=torch.int32, device=dev), 6, 8)
    rows, _ = ops.sparse_grad_rows(ops.build_feature_index(code), code.val, q, 8)
    want = ops.restore_rows(q, torch.float32)
    assert want[2, 32:64].isnan().all() and want[4, :32].isnan().all() and int(want.isnan().sum()) == 64
    assert torch.equal(rows[:6].isnan(), want.isnan()) and torch.equal(rows[:6].nan_to_num(), want.nan_to_num()) and not rows[6:].any()


# ---- streams, graphs, a run of them together ---------------------------------------------------------------------------

def test_another_stream(pkg, dev):
    ops = pkg.ops
    x = activations(512, 768, 19)
    want = ops.restore_rows(ops.quantize_rows(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.restore_rows(ops.quantize_rows(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_and_replayed_with_new_inputs(pkg, dev):
    """Write, pick a batch, and both weight gradients in one graph; every replay against the eager result."""
    ops = pkg.ops
    T, d, F, k = 192, 160, 64, 4
    x, g = activations(T, d, 20), activations(T, F, 21, torch.bfloat16)
    idx = torch.randint(0, T, (T,), device=dev)
    code = sparse_code(ops, T, F, k, 22, dev, True)

    def step():
        q = ops.quantize_rows(x)
        batch = ops.gather_rows(q, idx, torch.float32, 0.5)
        kept = ops.quantize_rows(batch)
        fi = ops.build_feature_index(code)
        return batch, ops.gemm_over_tokens(g, kept), ops.sparse_grad_rows(fi, code.val, kept, F, want_bias=True)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (30, 31, 32):
        x.copy_(activations(T, d, seed))
        idx.copy_(torch.randint(0, T, (T,), device=dev))
        code.val.copy_(torch.randn_like(code.val))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_two_graphs_replayed_in_turn(pkg, dev):
    """Two captures, each with its own temporary buffers, replayed in any order between eager work of the same operators."""
    ops = pkg.ops
    sizes = [(192, 160, 64, 4), (700, 96, 40, 9)]
    inputs = []
    for i, (T, d, F, k) in enumerate(sizes):
        inputs.append((activations(T, d, 40 + i), activations(T, F, 50 + i, torch.bfloat16), sparse_code(ops, T, F, k, 60 + i, dev, True)))

    def step(i):
        x, g, code = inputs[i]
        kept = ops.quantize_rows(x)
        fi = ops.build_feature_index(code)
        return (ops.restore_rows(kept, torch.float32), ops.gemm_over_tokens(g, kept),
                *ops.sparse_grad_rows(fi, code.val, kept, sizes[i][2], want_bias=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0), step(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for turn, i in enumerate((0, 1, 1, 0, 1, 0)):
        x, g, code = inputs[i]
        x.copy_(activations(*x.shape, 70 + turn))
        code.val.copy_(torch.randn_like(code.val))
        graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[i], step(i)):
            assert torch.equal(a, b)


# ---- refusals -------------------------------------------------------------------------------------------------

def test_refusals_on_the_device(pkg, dev):
    ops = pkg.ops
    x = activations(8, 64, 23)
    q = ops.quantize_rows(x)
    for bad in (x.double(), x.half(), x.to(torch.int32)):
        with pytest.raises(TypeError):
            ops.quantize_rows(bad)
    with pytest.raises(ValueError):
        ops.quantize_rows(x.t())                                             # values of a row lie apart
    with pytest.raises(ValueError):
        ops.quantize_rows(x[0])
    with pytest.raises(ValueError):
        ops.quantize_rows(x, out=torch.empty(7, pitch_of(64), dtype=torch.uint8, device=dev))
    with pytest.raises(ValueError):
        ops.quantize_rows(x, out=torch.empty(8, pitch_of(64) + 16, dtype=torch.uint8, device=dev))
    with pytest.raises(ValueError):
        ops.quantize_rows(x, out=torch.empty(8, pitch_of(64)).to(torch.uint8))    # on the CPU
    off = torch.empty(8 * pitch_of(64) + 1, dtype=torch.uint8, device=dev)[1:].view(8, -1)
    with pytest.raises(ValueError):
        ops.quantize_rows(x, out=off)                                        # not on a 16-byte boundary
    with pytest.raises(TypeError):
        ops.gather_rows(q, torch.zeros(2, dtype=torch.int32, device=dev))
    with pytest.raises(TypeError):
        ops.gather_rows(q, torch.zeros(2, dtype=torch.int64, device=dev), torch.float16)
    with pytest.raises(RuntimeError):
        ops.gather_rows(q, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.restore_rows(q, torch.float32, out=torch.empty(8, 65, device=dev))
    with pytest.raises(ValueError):
        ops.gather_rows(ops.quantize_rows(x[:0]), torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError):
        ops.gemm_over_tokens(torch.zeros(9, 8, dtype=torch.bfloat16, device=dev), q)
    with pytest.raises(TypeError):
        ops.gemm_over_tokens(x, q, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.gemm_over_tokens(x.half(), q)
    code = sparse_code(ops, 8, 6, 2, 24, dev)
    fi = ops.build_feature_index(code)
    with pytest.raises(ValueError):
        ops.sparse_grad_rows(fi, code.val, q, 7)
    with pytest.raises(ValueError):
        ops.sparse_grad_rows(fi, code.val[:-1].contiguous(), q, 6)
    with pytest.raises(ValueError):
        ops.sparse_grad_rows(fi, code.val, q, 6, out=torch.empty(6, 65, device=dev))
    with pytest.raises(ValueError):
        ops.sparse_grad_rows(fi, code.val, ops.quantize_rows(x[:0]), 6)      # slots of tokens, and no rows
    p = torch.zeros(6, 66, device=dev)
    odd = ops.quantize_rows(activations(8, 66, 25))
    with pytest.raises(RuntimeError):                                        # the Adam pass moves four values at a time
        ops.adam_step_sparse_rows(fi, code.val, odd, p, p.clone(), p.clone(), lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1)


def test_an_index_that_does_not_fit_is_refused(pkg, dev):
    ops = pkg.ops
    q = ops.quantize_rows(activations(8, 64, 23))
    code = sparse_code(ops, 8, 6, 2, 24, dev)
    fi = ops.build_feature_index(code)
    short, wide = code.val[:-1].contiguous(), torch.zeros(6, 64, device=dev)
    with pytest.raises(ValueError):
        ops.adam_step_sparse_rows(fi, short, q, wide, wide.clone(), wide.clone(), lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1)
    with pytest.raises(ValueError):
        ops.sparse_rows_grad_sq_nnz(fi, short, q, torch.zeros(2, dtype=torch.float64, device=dev))
    host = ops.FeatureIndex(fi.feat_ptr.cpu(), fi.feat_slot, fi.slot_tok)
    for call in (lambda: ops.sparse_grad_rows(host, code.val, q, 6),
                 lambda: ops.sparse_rows_grad_sq_nnz(host, code.val, q, torch.zeros(2, dtype=torch.float64, device=dev))):
        with pytest.raises(ValueError):
            call()
