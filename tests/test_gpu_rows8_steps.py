"""Train steps that keep what their backward pass reads in 8 bits, and the activation stream that holds rows in 8 bits.

The forward pass does not change (same loss, same selection, same bits); the weight gradients are those of the rows that 8 bits
hold.  Rows that 8 bits hold exactly therefore give the same gradients, which is checked to the bit where the order of
the sums is the same; for other rows the difference is bounded by half a step of every row that enters."""

import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def held(pkg, x):
    """The rows that 8 bits hold of x [..., d]."""
    flat = x.reshape(-1, x.shape[-1])
    return pkg.ops.restore_rows(pkg.ops.quantize_rows(flat), torch.float32).view(x.shape)


def half_steps(pkg, x):
    """[n, d] half the step of every value's block."""
    q = pkg.ops.quantize_rows(x)
    nb = -(-q.d // 32)
    field = q.data[:, 32 * nb : 33 * nb].to(torch.float64)
    return torch.where(field > 0, torch.exp2(field - 128), torch.zeros_like(field)).repeat_interleave(32, 1)[:, : q.d]


def autocast(amp):
    return torch.autocast("cuda", dtype=torch.bfloat16) if amp else contextlib.nullcontext()


def make_sae(pkg, dev, act_fn="topk", d=128, F=640, k=8, B=192, seed=0, dtype=torch.float32, x=None, **cfg):
    from lm_saes_amd import synthetic

    c = pkg.SAEConfig(hook_point_in="in", hook_point_out="out", d_model=d, expansion_factor=F / d, act_fn=act_fn, top_k=k,
                      norm_activation="inference", device="cuda", dtype=dtype, **cfg)
    sae = pkg.SparseAutoEncoder(c)
    host = synthetic.activations(B, d, 16, seed)
    synthetic.load_weights(sae, *[t.to(dev) for t in synthetic.sae_weights(d, F, host, seed)])
    if act_fn == "jumprelu":             # a new module's thresholds are memory as it came
        with torch.no_grad():
            sae.activation_function.log_jumprelu_threshold.fill_(-1.5)
    if cfg.get("use_glu_encoder"):
        with torch.no_grad():
            sae.W_E_glu.copy_(torch.randn(F, d, generator=torch.Generator().manual_seed(seed + 1)).t().to(dev) / d ** 0.5)
            sae.b_E_glu.zero_()
    x = held(pkg, host.to(dev)) if x is None else x
    label = synthetic.activations(B, d, 16, seed + 5).to(dev)
    return sae, {"in": x, "out": label, "tokens": torch.zeros(B, device=dev)}


def grads(model):
    return {n: p.grad.detach().clone() for n, p in model.named_parameters() if p.grad is not None}


class Sizes:
    """While installed, keeps for every gradient product over 8-bit rows the sum of its terms' magnitudes, as rows: what the
    rounding of its sums is relative to.  `encoder`: 8-bit inputs; `decoder`: 8-bit activations on the left."""

    def __init__(self, pkg, monkeypatch):
        self.encoder, self.decoder = [], []
        ops = pkg.ops
        sparse, dense = ops.sparse_grad_rows, ops.gemm_over_tokens

        def floats(t):
            return (ops.restore_rows(t, torch.float32) if isinstance(t, pkg.Rows8) else t.float()).abs()

        def sparse_grad_rows(fi, coef, rows, F, *a, **kw):
            if isinstance(rows, pkg.Rows8):
                self.encoder.append(sparse(fi, coef.abs(), ops.quantize_rows(floats(rows)), F)[0])
            return sparse(fi, coef, rows, F, *a, **kw)

        def gemm_over_tokens(left, right, *a, **kw):
            (self.decoder if isinstance(left, pkg.Rows8) else self.encoder).append(floats(left).t() @ floats(right))
            return dense(left, right, *a, **kw)

        monkeypatch.setattr(ops, "sparse_grad_rows", sparse_grad_rows)
        monkeypatch.setattr(ops, "gemm_over_tokens", gemm_over_tokens)


def close(got, want, size, terms, low):
    """Two sums of the same `terms` terms, each off by at most 2 terms 2^-24 of its terms' magnitudes (an addition rounds, or
    truncates inside a matrix instruction, once), each rounded to bf16 once more when `low`."""
    limit = 4.0 * terms * 2.0**-24 * size + (2.0 * 2.0**-8 * want.abs() * (1 + 2.0**-7) if low else 0.0)
    return ((got - want).abs() <= limit).all()


def run(model, batch, amp, keep, **kw):
    model.zero_grad(set_to_none=True)
    model.rows8_checkpoint = keep
    with autocast(amp):
        ctx = model.compute_loss(batch, **kw)
    ctx["loss"].backward()
    return ctx["loss"].detach().clone(), grads(model)


STEPS = [("topk", {}, {}), ("batchtopk", {}, {}), ("topk", {"sparsity_include_decoder_norm": True}, {}),
         ("topk", {"use_glu_encoder": True}, {}), ("topk", {}, {"sparsity_loss_type": "tanh", "l1_coefficient": 0.1}),
         ("jumprelu", {}, {"sparsity_loss_type": "tanh", "l1_coefficient": 0.1}), ("relu", {}, {})]


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("act_fn,cfg,kw", STEPS)
def test_rows_that_8_bits_hold_give_the_same_step(pkg, dev, monkeypatch, act_fn, cfg, kw, amp):
    """Loss and all gradients to the bit, but for the encoders' weights, whose sums may be formed in another order (and the
    decoder's where dense activations enter it from 8 bits, which is compared below)."""
    sae, batch = make_sae(pkg, dev, act_fn, **cfg)
    B = batch["in"].shape[0]
    loss, want = run(sae, batch, amp, False, **kw)
    sizes = Sizes(pkg, monkeypatch)
    loss8, got = run(sae, batch, amp, True, **kw)
    assert torch.equal(loss, loss8) and set(got) == set(want)
    encoders = [n for n in ("W_E", "W_E_glu") if n in want]
    assert len(sizes.encoder) == len(encoders)
    for n in want:
        if n in encoders:
            assert close(got[n], want[n], sizes.encoder[encoders.index(n)].t(), B, amp), n
        elif not (n == "W_D" and sizes.decoder):
            assert torch.equal(got[n], want[n]), n


LAYOUTS = [lambda x: x.t().contiguous().t(), lambda x: torch.cat([x, x], 1)[:, : x.shape[1]],
           lambda x: torch.stack([x, x], 2)[:, :, 0]]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("act_fn,cfg,kw", [STEPS[0], STEPS[3], STEPS[4], STEPS[5], STEPS[6]])
def test_inputs_of_any_strides(pkg, dev, act_fn, cfg, kw, amp, layout):
    """An fp32 batch that is a transposed or sliced view gives the step of its contiguous copy, with the option as without."""
    sae, batch = make_sae(pkg, dev, act_fn, **cfg)
    view = layout(batch["in"])
    assert not view.is_contiguous() and torch.equal(view, batch["in"])
    for keep in (False, True):
        loss, want = run(sae, batch, amp, keep, **kw)
        loss_v, got = run(sae, dict(batch, **{"in": view}), amp, keep, **kw)
        assert torch.equal(loss, loss_v) and set(got) == set(want)
        for n in want:
            assert torch.equal(got[n], want[n]), n
        sae.rows8_checkpoint = keep
        with autocast(amp):
            assert torch.equal(sae.encode(view), sae.encode(batch["in"]))


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("act_fn", ["topk", "batchtopk"])
def test_what_the_optimiser_is_handed(pkg, dev, act_fn, amp):
    """With HipAdam attached the encoder's gradient stays factored; its rows are 8-bit ones of the batch (of any batch: here
    one that 8 bits do not hold), everything else is to the bit what it is without, and so is the decoder's."""
    from lm_saes_amd import synthetic

    x = synthetic.activations(192, 128, 16, 3).to(dev)
    sae, batch = make_sae(pkg, dev, act_fn, x=x)
    opt = pkg.HipAdam(sae.get_parameters()[0]["params"], lr=1e-3, model=sae)
    parts = []
    for keep in (False, True):
        opt.zero_grad()
        sae.rows8_checkpoint = keep
        with autocast(amp):
            loss = sae.compute_loss(batch)["loss"]
        loss.backward()
        parts.append((loss.detach(), sae.W_E._sparse_grad, sae.W_D._sparse_grad, sae.b_D.grad.clone()))
    (la, ea, da, ba), (lb, eb, db, bb) = parts
    assert torch.equal(la, lb) and torch.equal(ba, bb) and torch.equal(da.coef, db.coef) and torch.equal(da.dense_operand, db.dense_operand)
    assert torch.equal(ea.coef, eb.coef) and torch.equal(ea.fi.feat_slot, eb.fi.feat_slot)
    assert isinstance(eb.dense_operand, pkg.Rows8) and torch.equal(eb.dense_operand.data, pkg.ops.quantize_rows(x).data)
    rows_a, bias_a = ea.dense()
    rows_b, bias_b = eb.dense()
    assert torch.equal(bias_a, bias_b)
    # |difference| <= sum of |coefficient| times (half a step + bf16's rounding of x under autocast) + the sums' own rounding
    off = half_steps(pkg, x) + (x.abs().double() * 2.0**-8 if amp else 0.0)
    slack = pkg.ops.sparse_grad_rows(ea.fi, ea.coef.abs(), off.float().contiguous(), 640)[0]
    size = pkg.ops.sparse_grad_rows(ea.fi, ea.coef.abs(), x.abs().contiguous(), 640)[0]
    assert ((rows_a - rows_b).abs() <= 1.01 * slack + 192 * 2.0**-22 * size).all()
    assert (rows_a - rows_b).abs().max() > 0
    before = sae.W_E.detach().clone()
    opt.step()
    assert torch.isfinite(sae.W_E).all() and not torch.equal(before, sae.W_E)


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("act_fn", ["topk", "jumprelu"])
def test_masked_tokens_give_the_gradients_nothing(pkg, dev, monkeypatch, act_fn, amp):
    """A padded batch: the step with masked tokens is the one without rows8_checkpoint, and other rows in their places change
    neither its loss nor its gradients (but for the order of the sums)."""
    sae, batch = make_sae(pkg, dev, act_fn)
    sae.jumprelu_sparse_route = False
    B, d = batch["in"].shape
    mask = torch.ones(B, device=dev)
    mask[B - 50:] = 0
    mask[7] = 0
    junk = batch["in"].clone()
    junk[mask == 0] = held(pkg, 30.0 * torch.randn(51, d, generator=torch.Generator(device=dev).manual_seed(2), device=dev))
    first = None
    for x in (batch["in"], junk):
        padded = dict(batch, mask=mask, **{"in": x})
        loss, want = run(sae, padded, amp, False)
        with monkeypatch.context() as patch:
            sizes = Sizes(pkg, patch)
            loss8, got = run(sae, padded, amp, True)
        assert torch.equal(loss, loss8)
        assert close(got["W_E"], want["W_E"], sizes.encoder[0].t(), B, amp)
        if first is None:
            first = loss8, got["W_E"]
        assert torch.equal(loss8, first[0])
        assert close(got["W_E"], first[1], sizes.encoder[0].t(), B, amp)


def test_gradients_against_differences_of_the_loss(pkg, dev):
    """The loss is a quadratic of W_E, and of W_D, as long as the selection stays: its central difference along any direction
    is the gradient's product with that direction, whatever the step.  The loss in 64 bits, from its formula, with the step's
    selection; the limit follows the rounding through the step: every sum of n terms is off by (n + 2) u of their magnitudes,
    u = 2^-23 for additions that round or, inside a matrix instruction, truncate."""
    u = 2.0**-23
    sae, batch = make_sae(pkg, dev)
    x, label = (batch[k].double() for k in ("in", "out"))
    B, d = x.shape
    sae.rows8_checkpoint = True
    sae.zero_grad(set_to_none=True)
    ctx = sae.compute_loss(batch)
    ctx["loss"].backward()
    on = (ctx["feature_acts"].detach() != 0).double()
    assert on.sum() > 0.5 * B * 8
    W_E, b_E, W_D, b_D = (p.detach().double() for p in (sae.W_E, sae.b_E, sae.W_D, sae.b_D))

    def loss(we, wd):
        recon = ((x @ we + b_E) * on) @ wd + b_D
        return ((recon - label) ** 2).sum(1).mean()

    # |error| of each quantity of the step
    acts, e_acts = (x @ W_E + b_E).abs() * on, (d + 3) * u * (x.abs() @ W_E.abs() + b_E.abs()) * on
    recon = ((x @ W_E + b_E) * on) @ W_D + b_D
    e_recon = e_acts @ W_D.abs() + (8 + 3) * u * (acts @ W_D.abs() + b_D.abs())
    g = 2.0 * (recon - label) / B
    e_g = 2.0 * (e_recon + u * (recon.abs() + label.abs())) / B + 4 * u * g.abs()
    dval = (g.abs() @ W_D.abs().t()) * on
    e_dval = (e_g @ W_D.abs().t()) * on + (d + 2) * u * dval
    e_WE = x.abs().t() @ e_dval + (B + 2) * u * (x.abs().t() @ dval)
    e_WD = e_acts.t() @ g.abs() + acts.t() @ e_g + (B + 2) * u * (acts.t() @ g.abs())
    rng = torch.Generator(device=dev).manual_seed(9)
    for name, grad, error in (("W_E", sae.W_E.grad.double(), e_WE), ("W_D", sae.W_D.grad.double(), e_WD)):
        directions = [grad / grad.norm()] + [torch.randn(grad.shape, generator=rng, device=dev, dtype=torch.float64) for _ in range(3)]
        one = torch.zeros(grad.shape, dtype=torch.float64, device=dev)
        one.view(-1)[grad.abs().reshape(-1).argmax()] = 1.0
        for v in directions + [one]:
            diff = ((loss(W_E + v, W_D) - loss(W_E - v, W_D)) if name == "W_E" else (loss(W_E, W_D + v) - loss(W_E, W_D - v))) / 2
            slack = 1e-12 * (loss(W_E + v, W_D) if name == "W_E" else loss(W_E, W_D + v))       # the difference's own, in 64 bits
            assert (diff - (grad * v).sum()).abs() <= (error * v.abs()).sum() + slack, name


def test_gradient_of_a_dense_decoder_against_differences(pkg, dev):
    """The same for the dense product over the token axis: acts @ W_D with activations that 8 bits hold, under a quadratic loss."""
    u = 2.0**-23
    sae, batch = make_sae(pkg, dev, "relu", d=128, F=640, B=77)
    sae.rows8_checkpoint = True
    acts = held(pkg, torch.rand(77, 640, generator=torch.Generator(device=dev).manual_seed(1), device=dev))
    label = batch["out"]
    timer = pkg.ops.KernelTimer()
    pkg.ops.set_kernel_timer(timer)
    try:
        (0.5 * (sae.decode(acts) - label).pow(2).sum()).backward()
    finally:
        pkg.ops.set_kernel_timer(None)
    assert "gemm_over_tokens" in timer.records and "rows8_quantize" in timer.records
    grad = sae.W_D.grad.double()
    W_D, b_D, A, y = sae.W_D.detach().double(), sae.b_D.detach().double(), acts.double(), label.double()
    loss = lambda w: 0.5 * (A @ w + b_D - y).pow(2).sum()                                       # noqa: E731
    out = A @ W_D + b_D
    e_out = (640 + 3) * u * (A @ W_D.abs() + b_D.abs()) + 2 * u * (out.abs() + y.abs())
    error = A.t() @ e_out + (77 + 2) * u * (A.t() @ (out - y).abs())
    rng = torch.Generator(device=dev).manual_seed(9)
    for v in [grad / grad.norm()] + [torch.randn(grad.shape, generator=rng, device=dev, dtype=torch.float64) for _ in range(3)]:
        diff = (loss(W_D + v) - loss(W_D - v)) / 2
        assert (diff - (grad * v).sum()).abs() <= (error * v.abs()).sum() + 1e-12 * loss(W_D + v)


@pytest.mark.parametrize("amp", [torch.float32, torch.bfloat16])
def test_a_trainer_over_held_inputs(pkg, dev, amp):
    """Trainer.fit with clipping: the same parameters to the bit with the inputs held as floats and in 8 bits."""
    from lm_saes_amd import synthetic

    d, F, B = 128, 512, 96
    finals = []
    for keep in (False, True):
        sae, _ = make_sae(pkg, dev, d=d, F=F, B=B)
        sae.rows8_checkpoint = keep
        stream = []
        for s in range(6):
            x = held(pkg, synthetic.activations(B, d, 16, s).to(dev))
            stream.append({"in": x, "out": x, "tokens": torch.zeros(B, device=dev)})
        trainer = pkg.Trainer(pkg.TrainerConfig(lr=1e-3, lr_warm_up_steps=2, lr_cool_down_steps=1, total_training_tokens=B * 6, amp_dtype=amp,
                                                l1_coefficient=None, log_frequency=3, k_warmup_steps=0, clip_grad_norm=0.05))
        trainer.fit(sae, stream)
        assert trainer.cur_step == 6
        finals.append([p.detach().clone() for p in sae.parameters()])
    for a, b in zip(*finals):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("lowp", [False, True])
def test_training_from_a_held_buffer_is_training_on_the_floats(pkg, dev, lowp):
    """A stream whose buffer holds records, steps that keep records, Adam that reads records: parameters and moments to the bit
    those of the same batches as floats, over several steps; with and without the gradient norm and clipping."""
    from lm_saes_amd import synthetic

    d, F, B = 128, 512, 96
    data = [{"in": synthetic.activations(150, d, 16, s).to(dev), "tokens": torch.zeros(150, device=dev)} for s in range(4)]
    finals = []
    for keep in (False, True):
        sae, _ = make_sae(pkg, dev, d=d, F=F, B=B, dtype=torch.bfloat16 if lowp else torch.float32)
        sae.rows8_checkpoint = keep
        opt = pkg.HipAdam(sae.get_parameters()[0]["params"], lr=1e-3, model=sae)
        floats = [dict(c, **{"in": held(pkg, c["in"])}) for c in data]
        kw = dict(buffer_size=300, buffer_shuffle_config=pkg.BufferShuffleConfig(perm_seed=2), override_dtype=torch.bfloat16)
        stream = pkg.ActivationBatchler(B, rows8={"in": d}, **kw).process(data) if keep else pkg.ActivationBatchler(B, **kw).process(floats)
        n = 0
        for i, batch in enumerate(stream):
            if batch["in"].shape[0] < B:
                continue
            opt.zero_grad()
            with autocast(not lowp):
                loss = sae.compute_loss(dict(batch, out=batch["in"].float()))["loss"]
            loss.backward()
            if i % 2:
                pkg.clip_grad_norm(sae.get_parameters()[0]["params"], 0.05)
            opt.step()
            n += 1
        assert n >= 4
        finals.append([p.detach().clone() for p in sae.parameters()] + [v for p in sae.parameters() for v in opt.state[p].values()])
    for a, b in zip(*finals):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dense_block", [True, False])
def test_aux_k_step(pkg, dev, monkeypatch, dense_block):
    """Both forms of the aux-k term (its stacked code reads every row twice)."""
    sae, batch = make_sae(pkg, dev, d=128, F=640, B=192)
    sae.aux_dense_block = dense_block
    dead = torch.zeros(640, dtype=torch.bool, device=dev)
    dead[::7] = True
    kw = dict(auxk_coefficient=0.25, k_aux=16, update_dead_statistics=lambda acts, mask, dims: dead)
    loss, want = run(sae, batch, True, False, **kw)
    assert sae._last_aux_route == ("dense" if dense_block else "sparse")
    sizes = Sizes(pkg, monkeypatch)
    loss8, got = run(sae, batch, True, True, **kw)
    assert torch.equal(loss, loss8) and len(sizes.encoder) == 1
    for n in want:
        if n == "W_E":      # a token enters twice, from either code; the dead features' block is added to either sum alike
            assert close(got[n], want[n], sizes.encoder[0].t() + want[n].abs(), 2 * 192 + 1, False), n
        else:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("amp", [False, True])
def test_dense_activations_enter_the_decoder_gradient_from_8_bits(pkg, dev, amp):
    sae, batch = make_sae(pkg, dev, "relu", d=128, F=640, B=192)
    sae.jumprelu_sparse_route = False
    loss, want = run(sae, batch, amp, False)
    loss8, got = run(sae, batch, amp, True)
    assert torch.equal(loss, loss8)
    with autocast(amp):
        ctx = sae.compute_loss(batch)
    acts = ctx["feature_acts"].detach()
    g = (2.0 * (ctx["reconstructed"].detach() - batch["out"]) / acts.shape[0]).double()
    off = half_steps(pkg, acts)
    size = acts.double().abs().t() @ g.abs()
    # half a step of the activations, plus bf16's roundings of g and of the result on both sides (or fp32's sums)
    limit = 1.01 * (off.t() @ g.abs()) + (4 * 2.0**-8 if amp else 2 * 192 * 2.0**-23) * size
    assert ((got["W_D"] - want["W_D"]).abs().double() <= limit).all() and (got["W_D"] - want["W_D"]).abs().max() > 0


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("B", [192, 77])
def test_encode_and_decode_products(pkg, dev, monkeypatch, amp, B):
    """The module's own products (any token count) hold their saved side in 8 bits when gradients are on."""
    sae, batch = make_sae(pkg, dev, "relu", d=128, F=640, B=B)
    x = batch["in"]
    sae.zero_grad(set_to_none=True)
    outs, gs, sizes = [], [], None
    for keep in (False, True):
        sae.rows8_checkpoint = keep
        sizes = Sizes(pkg, monkeypatch) if keep else None
        sae.zero_grad(set_to_none=True)
        with autocast(amp):
            acts = sae.encode(x)
            held_acts = held(pkg, acts.detach().float()).to(acts.dtype).requires_grad_(True)
            out = sae.decode(held_acts)
        g = torch.randn(acts.shape, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(acts.dtype)
        torch.autograd.backward([acts, out], [g, g[:, :128].contiguous().to(out.dtype)])
        outs.append((acts.detach(), out.detach(), held_acts.grad))
        gs.append(grads(sae))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert close(gs[1]["W_E"], gs[0]["W_E"], sizes.encoder[0].t(), B, amp)
    if sizes.decoder:                                        # enough of the activations are not zero: the dense product
        assert close(gs[1]["W_D"], gs[0]["W_D"], sizes.decoder[0], B, amp)
    else:
        assert torch.equal(gs[1]["W_D"], gs[0]["W_D"])
    sae.rows8_checkpoint = True
    timer = pkg.ops.KernelTimer()
    pkg.ops.set_kernel_timer(timer)
    try:
        with torch.no_grad(), autocast(amp):
            sae.encode(x)
        assert "rows8_quantize" not in timer.records
        with autocast(amp):
            sae.encode(x)
        assert "rows8_quantize" in timer.records
    finally:
        pkg.ops.set_kernel_timer(None)


def test_a_step_holds_less_between_its_passes(pkg, dev):
    sae, batch = make_sae(pkg, dev, "relu", d=256, F=8192, B=1024)
    sae.jumprelu_sparse_route = False
    used = []
    for keep in (False, True):
        sae.zero_grad(set_to_none=True)
        sae.rows8_checkpoint = keep
        torch.cuda.synchronize()
        with autocast(True):
            sae.compute_loss(batch, return_aux_data=False).backward()          # operands that outlive the step are made here
        sae.zero_grad(set_to_none=True)
        start = torch.cuda.memory_allocated()
        with autocast(True):
            loss = sae.compute_loss(batch, return_aux_data=False)
        used.append(torch.cuda.memory_allocated() - start)
        loss.backward()
    # bf16 activations [B, F] and inputs [B, d] become records
    saved = 1024 * (2 * 8192 - pkg.ops.rows8_pitch(8192) + 2 * 256 - pkg.ops.rows8_pitch(256))
    assert used[0] - used[1] >= 0.95 * saved, used


# ---- the variants -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("amp", [False, True])
def test_crosscoder_step(pkg, dev, monkeypatch, amp):
    H, d, F, k, B = 2, 96, 512, 6, 128
    hooks = [f"h{i}" for i in range(H)]
    torch.manual_seed(0)
    cc = pkg.Crosscoder(pkg.CrosscoderConfig(hook_points=hooks, d_model=d, expansion_factor=F / d, act_fn="topk", top_k=k,
                                             norm_activation="inference", device="cuda", dtype=torch.float32))
    g = torch.Generator(device=dev).manual_seed(1)
    with torch.no_grad():
        for p in cc.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.1)
    x = held(pkg, torch.randn(B, H, d, generator=g, device=dev).view(B, H * d)).view(B, H, d)
    batch = {h: x[:, i].contiguous() for i, h in enumerate(hooks)} | {"tokens": torch.zeros(B, device=dev)}
    loss, want = run(cc, batch, amp, False)
    sizes = Sizes(pkg, monkeypatch)
    loss8, got = run(cc, batch, amp, True)
    assert torch.equal(loss, loss8) and len(sizes.encoder) == 1
    for n in want:
        if n == "W_E":
            assert close(got[n], want[n], sizes.encoder[0].view(F, H, d).permute(1, 2, 0), H * B, False), n
        else:
            assert torch.equal(got[n], want[n]), n
    opt = pkg.HipAdam(cc.get_parameters()[0]["params"], lr=1e-3, model=cc)
    opt.zero_grad()
    with autocast(amp):
        cc.compute_loss(batch)["loss"].backward()
    assert isinstance(cc.W_E._sparse_grad.dense_operand, pkg.Rows8) and cc.W_E._sparse_grad.dense_operand.shape == (B, H * d)
    opt.step()
    assert all(torch.isfinite(p).all() for p in cc.parameters())


@pytest.mark.parametrize("act_fn", ["topk", "layertopk", "jumprelu"])
@pytest.mark.parametrize("amp", [False, True])
def test_clt_step(pkg, dev, monkeypatch, act_fn, amp):
    """A layer's encoder reads its stretch of the one feature index that serves all layers."""
    L, d, F, k, B = 3, 64, 256, 5, 128
    hin, hout = [f"i{l}" for l in range(L)], [f"o{l}" for l in range(L)]
    clt = pkg.CrossLayerTranscoder(pkg.CLTConfig(hook_points_in=hin, hook_points_out=hout, d_model=d, expansion_factor=F / d, act_fn=act_fn,
                                                 top_k=k, norm_activation="inference", device="cuda", dtype=torch.float32))
    g = torch.Generator(device=dev).manual_seed(2)
    with torch.no_grad():
        for n, p in clt.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.1 if "log" not in n else torch.full(p.shape, -2.0, device=dev))
    x = held(pkg, torch.randn(B, L, d, generator=g, device=dev))
    batch = {h: x[:, l].contiguous() for l, h in enumerate(hin)} | {h: torch.randn(B, d, generator=g, device=dev) for h in hout}
    batch["tokens"] = torch.zeros(B, device=dev)
    loss, want = run(clt, batch, amp, False)
    sizes = Sizes(pkg, monkeypatch)
    loss8, got = run(clt, batch, amp, True)
    assert torch.equal(loss, loss8) and len(sizes.encoder) == L
    for n in want:
        if n == "W_E":
            assert close(got[n], want[n], torch.stack(sizes.encoder).permute(0, 2, 1), B, amp), n
        elif not (sizes.decoder and n.startswith("W_D")):       # dense activations enter that gradient from 8 bits
            assert torch.equal(got[n], want[n]), n
    opt = pkg.HipAdam(clt.get_parameters()[0]["params"], lr=1e-3, model=clt)
    opt.zero_grad()
    with autocast(amp):
        clt.compute_loss(batch)["loss"].backward()
    opt.step()
    assert all(torch.isfinite(p).all() for p in clt.parameters())


@pytest.mark.parametrize("rotary", [False, True])
def test_lorsa_step_forms_its_mixing_again(pkg, dev, rotary):
    """Of inputs that 8 bits hold the mixing formed again in the backward pass is the one of the forward pass: every gradient to
    the bit, with less held between the passes; of others it is the mixing of the rows that 8 bits hold."""
    d, F, h, s, b, k = 128, 256, 4, 64, 4, 8
    kw = dict(positional_embedding_type="rotary" if rotary else "none", rotary_dim=32)
    lorsa = pkg.LowRankSparseAttention(pkg.LorsaConfig(
        hook_point_in="in", hook_point_out="out", d_model=d, expansion_factor=F / d, n_qk_heads=h, d_qk_head=32, n_ctx=s, top_k=k,
        act_fn="topk", norm_activation="inference", device="cuda", dtype=torch.float32, **kw))
    g = torch.Generator(device=dev).manual_seed(6)
    with torch.no_grad():
        for p in lorsa.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.1)
    raw = torch.randn(b, s, d, generator=g, device=dev)
    batch = {"in": held(pkg, raw), "out": torch.randn(b, s, d, generator=g, device=dev), "tokens": torch.zeros(b, s, device=dev)}
    assert lorsa.rows8_checkpoint is False
    with autocast(True):
        assert lorsa._mix_kernel_eligible(batch["in"])
    loss, want = run(lorsa, batch, True, False)
    loss8, got = run(lorsa, batch, True, True)
    assert torch.equal(loss, loss8) and set(got) == set(want)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    used = []
    for keep in (False, True):
        lorsa.rows8_checkpoint = keep
        start = torch.cuda.memory_allocated()
        with autocast(True):
            z = lorsa.compute_hidden_pre(raw)
        used.append(torch.cuda.memory_allocated() - start)
        out = torch.autograd.grad(z, [lorsa.W_Q, lorsa.W_V], torch.ones_like(z))
        del z
    with autocast(True):
        z = lorsa.compute_hidden_pre(held(pkg, raw))
    for a, c in zip(out, torch.autograd.grad(z, [lorsa.W_Q, lorsa.W_V], torch.ones_like(z))):
        assert torch.equal(a, c)                            # what the 8-bit run formed from `raw`
    with autocast(True):
        z = lorsa.compute_hidden_pre(raw)
    with torch.no_grad():
        lorsa.W_K.mul_(1.5)
    with pytest.raises(RuntimeError, match="changed between the two passes"):
        z.sum().backward()
    saved = b * s * (2 * d - pkg.ops.rows8_pitch(d) + 2 * (2 * h * 32 + F))     # x, q, k, v in bf16; the mixing itself is the output
    assert used[0] - used[1] >= 0.9 * saved, used


@pytest.mark.parametrize("T", [60, 300, 330, 700])
def test_a_stretch_of_an_index(pkg, dev, T):
    """Gradient rows of features in the middle of an index: neither what lies before nor behind them is touched or read."""
    ops = pkg.ops
    F, k, d = 90, 9, 132
    g = torch.Generator(device=dev).manual_seed(3)
    idx = torch.rand(T, F, generator=g, device=dev).topk(k, 1).indices.sort(1).values.to(torch.int32).reshape(-1).contiguous()
    val = torch.randn(T * k, generator=g, device=dev)
    code = ops.SparseCode(idx, val, torch.arange(T, device=dev) * k, torch.full((T,), k, dtype=torch.int32, device=dev), T, F)
    fi = ops.build_feature_index(code)
    q = ops.quantize_rows(torch.randn(T, d, generator=g, device=dev))
    whole, bias = ops.sparse_grad_rows(fi, val, q, F, want_bias=True)
    size, _ = ops.sparse_grad_rows(fi, val.abs(), ops.quantize_rows(ops.restore_rows(q, torch.float32).abs()), F)
    for lo, hi in ((0, 30), (30, 60), (60, 90), (41, 42), (89, 90)):
        part = ops.FeatureIndex(fi.feat_ptr[lo : hi + 1], fi.feat_slot, fi.slot_tok)
        frame = torch.full((hi - lo + 2, d), 7.0, device=dev)
        rows, b = ops.sparse_grad_rows(part, val, q, hi - lo, want_bias=True, out=frame[1:-1])
        # the same terms, which the number of features may let in another order
        assert close(rows, whole[lo:hi], size[lo:hi], T, False) and torch.equal(b, bias[lo:hi]) and (frame[0] == 7).all() and (frame[-1] == 7).all()


@pytest.mark.parametrize("T,F,k,d", [(1100, 90, 9, 132), (2000, 300, 24, 40), (1500, 64, 40, 1030), (60, 90, 9, 132)])
def test_a_stretch_whose_slots_are_counted(pkg, dev, T, F, k, d):
    """With its largest number of slots said, a stretch gives the bits of the index that begins with it; with too few said the
    rows are NaN (right, where one launch does it all), and nothing beside them is touched."""
    ops = pkg.ops
    g = torch.Generator(device=dev).manual_seed(5)
    score = torch.rand(T, F, generator=g, device=dev)
    score[:, F // 2] = 2.0                                                     # a feature of every token
    idx = score.topk(k, 1).indices.sort(1).values.to(torch.int32).reshape(-1).contiguous()
    val = torch.randn(T * k, generator=g, device=dev)
    code = ops.SparseCode(idx, val, torch.arange(T, device=dev) * k, torch.full((T,), k, dtype=torch.int32, device=dev), T, F)
    fi = ops.build_feature_index(code)
    ptr = fi.feat_ptr.tolist()
    q = ops.quantize_rows(torch.randn(T, d, generator=g, device=dev))
    lib = pkg._lib.load()
    for lo, hi in ((0, F), (0, F // 3), (F // 3, F - 2), (F // 2, F // 2 + 1), (F - 1, F)):
        used, n = ptr[hi] - ptr[lo], hi - lo
        part = ops.FeatureIndex(fi.feat_ptr[lo : hi + 1], fi.feat_slot, fi.slot_tok)
        front = ops.FeatureIndex(part.feat_ptr - ptr[lo], torch.roll(fi.feat_slot, -ptr[lo]), fi.slot_tok)
        for said in (used, used + 1, used + 777, 10**9):
            frame = torch.full((n + 2, d), 7.0, device=dev)
            rows, b = ops.sparse_grad_rows(part, val, q, n, want_bias=True, out=frame[1:-1], max_slots=said)
            want, b0 = ops.sparse_grad_rows(front, val, q, n, want_bias=True, max_slots=said)
            assert torch.equal(rows, want) and torch.equal(b, b0) and (frame[0] == 7).all() and (frame[-1] == 7).all()
        frame = torch.full((n + 2, d), 7.0, device=dev)
        rows, b = ops.sparse_grad_rows(part, val, q, n, want_bias=True, out=frame[1:-1], max_slots=used - 1)
        if lib.sae_rows8_grad_rows_workspace_bytes(T, used - 1, n, d):
            assert rows.isnan().all() and b.isnan().all()
        else:
            assert torch.isfinite(rows).all() and torch.equal(b, b0)
        assert (frame[0] == 7).all() and (frame[-1] == 7).all()
    with pytest.raises(ValueError):
        ops.sparse_grad_rows(fi, val, q, F, max_slots=-1)


@pytest.mark.parametrize("act_fn", ["topk", "batchtopk", "layertopk"])
@pytest.mark.parametrize("granule", [True, False])
def test_a_layer_pays_for_its_own_slots(pkg, dev, monkeypatch, act_fn, granule):
    """The cross-layer transcoder says how many slots a layer has at most: all there are in it, and no more than one layer's share
    where every layer selects by itself."""
    L, d, F, k, B = 4, 64, 256, 6, 1200
    hin, hout = [f"i{l}" for l in range(L)], [f"o{l}" for l in range(L)]
    clt = pkg.CrossLayerTranscoder(pkg.CLTConfig(hook_points_in=hin, hook_points_out=hout, d_model=d, expansion_factor=F / d, act_fn=act_fn,
                                                 top_k=k, norm_activation="inference", device="cuda", dtype=torch.float32))
    clt.granule_select = granule
    g = torch.Generator(device=dev).manual_seed(2)
    with torch.no_grad():
        for p in clt.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.1)
    x = held(pkg, torch.randn(B, L, d, generator=g, device=dev))
    batch = {h: x[:, l].contiguous() for l, h in enumerate(hin)} | {h: torch.randn(B, d, generator=g, device=dev) for h in hout}
    batch["tokens"] = torch.zeros(B, device=dev)
    said, plain = [], pkg.ops.sparse_grad_rows

    def sparse_grad_rows(fi, coef, rows, F, *a, **kw):
        if isinstance(rows, pkg.Rows8):
            said.append((int(fi.feat_ptr[-1] - fi.feat_ptr[0]), kw["max_slots"]))
        return plain(fi, coef, rows, F, *a, **kw)

    monkeypatch.setattr(pkg.ops, "sparse_grad_rows", sparse_grad_rows)
    _, got = run(clt, batch, True, True)
    assert len(said) == L and all(used <= most for used, most in said) and all(torch.isfinite(v).all() for v in got.values())
    if act_fn != "layertopk":
        assert all(most <= B * k for _, most in said)


def make_variant(pkg, dev, kind):
    """A small crosscoder, cross-layer transcoder or Lorsa, and a batch of it."""
    n, d, F, B = 2, 64, 256, 128
    common = dict(d_model=d, expansion_factor=F / d, act_fn="topk", top_k=5, norm_activation="inference", device="cuda", dtype=torch.float32)
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(n, B, d, generator=g, device=dev)
    hin, hout = [f"i{i}" for i in range(n)], [f"o{i}" for i in range(n)]
    if kind == "crosscoder":
        model = pkg.Crosscoder(pkg.CrosscoderConfig(hook_points=hin, **common))
    elif kind == "clt":
        model = pkg.CrossLayerTranscoder(pkg.CLTConfig(hook_points_in=hin, hook_points_out=hout, **common))
    else:
        model = pkg.LowRankSparseAttention(pkg.LorsaConfig(hook_point_in="i0", hook_point_out="o0", n_qk_heads=4, d_qk_head=32, n_ctx=64,
                                                           positional_embedding_type="none", rotary_dim=32, **common))
        x = x.view(2, 2, 64, d)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.1)
    return model, dict(zip(hin, x)) | dict(zip(hout, x.flip(0))) | {"tokens": torch.zeros(x.shape[1:-1], device=dev)}


KINDS = list(range(len(STEPS))) + ["aux", "dense", "crosscoder", "clt"]


@pytest.mark.parametrize("kind,amp", [(k, amp) for k in KINDS for amp in (False, True)] + [("lorsa", True)])
def test_records_are_written_for_a_backward_pass_only(pkg, dev, kind, amp):
    """A loss without gradients (an evaluation, a search over scales) is that of the model without the option, and writes nothing."""
    kw = {}
    if kind in ("crosscoder", "clt", "lorsa"):
        model, batch = make_variant(pkg, dev, kind)
    elif kind == "aux":
        model, batch = make_sae(pkg, dev)
        dead = torch.arange(640, device=dev) % 3 == 0
        kw = dict(auxk_coefficient=0.1, k_aux=16, update_dead_statistics=lambda *a, **k: dead)
    elif kind == "dense":
        model, batch = make_sae(pkg, dev, "relu")
        model.jumprelu_sparse_route = False
    else:
        act_fn, cfg, kw = STEPS[kind]
        model, batch = make_sae(pkg, dev, act_fn, **cfg)
    timer = pkg.ops.KernelTimer()
    pkg.ops.set_kernel_timer(timer)
    try:
        losses = []
        for keep, mode in ((False, torch.no_grad), (True, torch.no_grad), (True, torch.inference_mode)):
            model.rows8_checkpoint = keep
            with mode(), autocast(amp):
                losses.append(model.compute_loss(batch, **kw)["loss"].clone())
        assert torch.equal(losses[0], losses[1]) and torch.equal(losses[0], losses[2])
        assert "rows8_quantize" not in timer.records
        with autocast(amp):
            loss = model.compute_loss(batch, **kw)["loss"]
        assert torch.equal(loss.detach(), losses[0]) and "rows8_quantize" in timer.records
        loss.backward()
    finally:
        pkg.ops.set_kernel_timer(None)


# ---- the stream --------------------------------------------------------------------------------------------------

def test_records_made_on_either_side_are_the_same(pkg, dev):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = (torch.randn(50, 77) * torch.exp(3 * torch.randn(50, 1))).to(dtype)
        x[3, 5], x[4, 70], x[5] = float("inf"), float("nan"), 0.0
        a, b = pkg.rows8_pack(x), pkg.rows8_pack(x.to(dev))
        assert torch.equal(a, b.cpu())
        for to in (torch.float32, torch.bfloat16, torch.float16):
            u, v = pkg.rows8_unpack(a, 77, to, 0.7), pkg.rows8_unpack(b, 77, to, 0.7)
            assert v.dtype == to and torch.equal(u.isnan(), v.cpu().isnan()) and torch.equal(u.nan_to_num(), v.cpu().nan_to_num())


def test_no_rows_on_the_gpu(pkg, dev):
    for shape in ((0, 40), (2, 0, 33), (0, 1)):
        data = pkg.rows8_pack(torch.zeros(shape, device=dev))
        assert data.is_cuda and tuple(data.shape) == (*shape[:-1], pkg.ops.rows8_pitch(shape[-1]))
        assert tuple(pkg.rows8_unpack(data, shape[-1], torch.bfloat16).shape) == shape


def test_cached_stream_of_records_on_the_gpu_equals_the_cpu_stream(pkg, dev, tmp_path):
    hooks = ["in", "out"]
    g = torch.Generator().manual_seed(4)

    def samples():
        for i in range(9):
            t = torch.arange(16)[None] + 100 * i
            yield {"in": torch.randn(1, 16, 70, generator=g), "out": torch.randn(1, 16, 64, generator=g), "tokens": t,
                   "mask": (t % 3 != 0).long(), "attention_mask": torch.ones_like(t)}

    pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path), hook_points=hooks, n_samples_per_chunk=2, row_format="rows8")
                         ).process(samples())
    for kw in ({}, {"override_dtype": torch.float32}, {"override_dtype": torch.float16}, {"dtype": torch.float32}):
        for rows8 in (False, True):
            base = dict(batch_size=20, buffer_size=60, buffer_shuffle_config=pkg.BufferShuffleConfig(perm_seed=5), rows8=rows8, **kw)
            cpu = list(pkg.cached_activation_stream(tmp_path, hooks, device="cpu", **base))
            gpu = list(pkg.cached_activation_stream(tmp_path, hooks, device="cuda", **base))
            assert len(cpu) == len(gpu) > 3
            for a, b in zip(cpu, gpu):
                for hp in hooks:
                    assert b[hp].is_cuda and a[hp].dtype == b[hp].dtype and torch.equal(a[hp], b[hp].cpu())
                assert torch.equal(a["tokens"], b["tokens"].cpu())


def test_rows_that_arrive_on_another_device_than_the_buffer(pkg, dev):
    """A buffer lies where its first rows did; later ones may come from the other side."""
    x = torch.randn(90, 70, generator=torch.Generator().manual_seed(4))
    want = pkg.rows8_unpack(pkg.rows8_pack(x), 70, torch.float32)
    for first, second in ((torch.device("cpu"), dev), (dev, torch.device("cpu"))):
        chunks = [{"in": x[:40].to(first)}, {"in": x[40:].to(second)}]
        got = torch.cat([b["in"] for b in pkg.ActivationBatchler(30, buffer_size=100, rows8={"in": 70}).process(chunks)])
        assert got.device.type == first.type and got.dtype == torch.float32 and torch.equal(got.cpu(), want)


def test_chunks_of_several_types_and_forms_on_the_gpu(pkg, dev, tmp_path):
    """What a chunk comes out as is its own, though the reader is ahead of it; a file that is refused ends the pass behind the
    chunks in front of it, as on the CPU."""
    def write(path, parts):
        for i, (dtype, form) in enumerate(parts):
            t = torch.arange(16)[None]
            x = torch.randn(1, 16, 40, generator=torch.Generator().manual_seed(i)).to(dtype)
            x[0, 3, 3] = 6e4 if dtype == torch.float16 else 1e5
            pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(path), hook_points=["h"], row_format=form)).process(
                [{"h": x, "tokens": t, "mask": torch.ones_like(t), "attention_mask": torch.ones_like(t)}], start_shard=i)

    f32, bf16, f16 = torch.float32, torch.bfloat16, torch.float16
    for n, parts in enumerate(([(bf16, "rows8"), (f16, "rows8"), (f32, "rows8")], [(f32, "float"), (bf16, "rows8"), (f16, "rows8")])):
        write(tmp_path / str(n), parts)
        for dtype in (None, f32):
            cpu, gpu = (pkg.CachedActivationLoader({"h": tmp_path / str(n) / "h"}, device=d, dtype=dtype) for d in ("cpu", "cuda"))
            for _ in range(2):
                a, b = list(cpu.process()), list(gpu.process())
                assert len(a) == len(b) == 3
                for u, v, (written, _form) in zip(a, b, parts):
                    assert u["h"].dtype == v["h"].dtype == (dtype or written) and torch.equal(u["h"], v["h"].cpu())
    write(tmp_path / "refused", [(f32, "rows8"), (f32, "rows8"), (f32, "float")])
    for d in ("cpu", "cuda"):
        it = pkg.CachedActivationLoader({"h": tmp_path / "refused" / "h"}, device=d).process()
        assert next(it)["h"].dtype == next(it)["h"].dtype == f32
        with pytest.raises(ValueError, match="float rows after"):
            next(it)


def test_a_stream_of_floats_holds_floats_on_the_gpu(pkg, dev, tmp_path):
    """Rows of a float file in front of 8-bit ones reach the batches as they are, however far ahead the reader is."""
    for i, form in enumerate(("float", "rows8", "rows8")):
        t = torch.arange(16)[None] + 100 * i
        x = torch.randn(1, 16, 40, generator=torch.Generator().manual_seed(i))
        pkg.ActivationWriter(pkg.ActivationWriterConfig(cache_dir=str(tmp_path), hook_points=["h"], row_format=form)).process(
            [{"h": x, "tokens": t, "mask": torch.ones_like(t), "attention_mask": torch.ones_like(t)}], start_shard=i)
    kw = dict(batch_size=8, buffer_size=24, buffer_shuffle_config=pkg.BufferShuffleConfig(perm_seed=7))
    cpu, gpu = (list(pkg.cached_activation_stream(tmp_path, ["h"], device=d, **kw)) for d in ("cpu", "cuda"))
    assert len(cpu) == len(gpu) == 6
    for a, b in zip(cpu, gpu):
        assert torch.equal(a["tokens"], b["tokens"].cpu()) and torch.equal(a["h"], b["h"].cpu())
    x = torch.randn(1, 16, 40, generator=torch.Generator().manual_seed(0))[0]
    rows = torch.cat([b["h"].cpu() for b in gpu])[torch.cat([b["tokens"].cpu() for b in gpu]).reshape(-1).argsort()]
    assert torch.equal(rows[:16], x)
