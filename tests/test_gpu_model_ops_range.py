"""The operators of the model over ranges that ordinary sizes and values do not reach: large soft caps, long rows and lists, what
autograd has to be told, limits of the index arithmetic.

Bounds are those of the arithmetic, as in test_gpu_model_ops."""
import math

import pytest
import torch

from test_gpu_model_ops import BF, EPS, F32, _check_table_gradient, _gen, _loss_problem, _qk_problem, _within

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------------------------------------------- cross entropy
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows, vocab", [(40, 1000), (70, 70001), (2, 131072)])
@pytest.mark.parametrize("softcap", [50.0, 1e4, 1e6, 1e20, 1e30])
def test_cross_entropy_with_large_caps(dev, dtype, rows, vocab, softcap):
    """A capped logit is off by rounded operations on itself, whatever the cap: x / cap by two products with rounded factors (3), its
    exponential and what follows from it at most 21 units of 2^-24 of the logit where |x| >= 0.3 cap, below that a polynomial (6)."""
    from dion_amd import cross_entropy, cross_entropy_with_grad
    from oracle import model_ops as O

    logits, targets = _loss_problem(rows, vocab, dtype, seed=rows)
    targets[0] = 0
    x, t = logits.to(dev), targets.to(dev)
    live = targets != -100
    losses, lse = O.cross_entropy(logits, targets, softcap=softcap)
    z = O.capped(logits.double(), softcap)
    off = 24 * EPS * logits.double().abs().clamp(max=softcap)
    dlse = (vocab / 64 + 44) * 2 * EPS + 2 * EPS * lse.abs() + off.max(-1).values
    at = targets.clamp(min=0)[:, None]
    slack = torch.where(live, dlse + off.gather(-1, at)[:, 0] + 2 * EPS * z.gather(-1, at)[:, 0].abs(), 0.0)
    far = (z - lse[:, None]).abs().clamp(max=200)
    dslack = torch.exp(z - lse[:, None]) * (dlse[:, None] + off + (2 * far + 28) * EPS)
    dslack.scatter_add_(-1, at, torch.full_like(lse, 24 * EPS)[:, None])

    _within(cross_entropy(x, t, reduction="none", softcap=softcap), losses, slack, "losses")
    want = O.cross_entropy_grad(logits, targets, 1.0, softcap=softcap)
    loss, dx = cross_entropy_with_grad(x, t, reduction="sum", softcap=softcap)
    _within(loss, losses.sum(), slack.sum(), "sum")
    _within(dx, want, dslack + 4 * EPS * want.abs(), "gradient")
    leaf = x.clone().requires_grad_(True)
    cross_entropy(leaf, t, reduction="sum", softcap=softcap).backward()
    _within(leaf.grad, want, dslack + 4 * EPS * want.abs(), "autograd")


def test_cross_entropy_refuses_a_cap_that_is_no_float(dev):
    """A cap that float32 rounds to zero is no missing one."""
    from dion_amd import cross_entropy, cross_entropy_with_grad
    from dion_amd._lib import DionAmdError

    z, t = torch.randn(3, 10, device=dev), torch.zeros(3, dtype=torch.long, device=dev)
    for cap in (1e-50, -1e-50, 1e50, math.nan):
        for call in (cross_entropy, cross_entropy_with_grad):
            with pytest.raises(DionAmdError, match="positive number"):
                call(z, t, softcap=cap)


def test_negated_upstream_gradient_of_the_loss(dev):
    """The upstream gradient may be a tensor whose memory holds the negative of its values."""
    from dion_amd import cross_entropy

    z, t = torch.randn(3, 10, device=dev), torch.tensor([1, 4, 9], device=dev)
    for reduction, up in (("mean", torch.randn((), device=dev)), ("none", torch.randn(3, device=dev))):
        negated = torch.complex(torch.zeros_like(up), -up).conj().imag
        assert negated.is_neg() and torch.equal(negated, up)
        grads = []
        for d in (up, negated):
            leaf = z.clone().requires_grad_(True)
            cross_entropy(leaf, t, reduction=reduction).backward(d)
            grads.append(leaf.grad)
        assert torch.equal(*grads)


# ------------------------------------------------------------------------------------------------------------- autograd
def test_given_table_gradient_counts_as_modified(dev):
    from dion_amd import embedding_backward

    grad, tokens = torch.randn(3, 8, device=dev), torch.tensor([1, 4, 1], device=dev)
    for accumulate in (False, True):
        out, leaf = torch.randn(10, 8, device=dev), torch.randn(10, 8, device=dev, requires_grad=True)
        loss = (leaf * out).sum()
        embedding_backward(grad, tokens, 10, out=out, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_rotation_tables_that_want_a_gradient_are_refused(dev):
    import dion_amd as A
    from dion_amd._lib import DionAmdError

    x = torch.randn(1, 3, 2, 8, device=dev)
    cos, sin = A.rope_tables(3, 8, device=dev)
    for tables in ((cos.clone().requires_grad_(True), sin), (cos, sin.clone().requires_grad_(True))):
        with pytest.raises(DionAmdError, match="cos and sin are constants"):
            A.qk_norm_rope(x, x, *tables)
        with torch.no_grad():
            q, _ = A.qk_norm_rope(x, x, *tables)
        assert torch.equal(q, A.qk_norm_rope(x, x, cos, sin)[0])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(sin, torch.ones_like(sin))
        with pytest.raises(DionAmdError, match="forward mode"):
            A.qk_norm_rope(x, x, cos, dual)


def test_tangents_are_refused_by_the_gradients(dev):
    """What the gradients would have to do with a tangent they do not: none is dropped without a word."""
    import dion_amd as A
    from dion_amd._lib import DionAmdError

    w, t = torch.randn(3, 8, device=dev), torch.tensor([1, 4, 1], device=dev)
    x = torch.randn(1, 3, 2, 8, device=dev)
    cos, sin = A.rope_tables(3, 8, device=dev)
    gain = torch.rand(8, device=dev)
    table, q, z = (a.clone().requires_grad_(True) for a in (torch.randn(5, 8, device=dev), x, w))
    with torch.autograd.forward_ad.dual_level():
        dual = lambda a: torch.autograd.forward_ad.make_dual(a.detach().clone(), torch.ones_like(a))  # noqa: E731
        for call in (lambda: A.embedding_backward(dual(w), t, 5), lambda: A.embedding_backward(w, t, 5, out=dual(table), accumulate=True),
                     lambda: A.qk_norm_rope_backward(dual(x), x, x, x, cos, sin), lambda: A.qk_norm_rope_backward(x, x, x, dual(x), cos, sin),
                     lambda: A.qk_norm_rope_backward(x, x, x, x, dual(cos), sin),
                     lambda: A.qk_norm_rope_backward(x, x, x, x, cos, sin, q_gain=dual(gain), k_gain=gain),
                     lambda: A.cross_entropy_with_grad(dual(w), t), lambda: A.cross_entropy_with_grad(dual(w), t, inplace=True)):
            with pytest.raises(DionAmdError, match="forward mode"):
                call()
        for out, leaf in ((A.embedding(table, t), table), (A.qk_norm_rope(q, x, cos, sin)[0], q), (A.cross_entropy(z, t, reduction="none"), z)):
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(out, leaf, dual(out))


def test_exceptions_keep_their_type(dev):
    """No memory is torch.OutOfMemoryError, as of any operator; an exception of a hook on saved tensors is that exception."""
    import dion_amd as A

    w, t = torch.randn(10, 8, device=dev, requires_grad=True), torch.tensor([1, 4, 1], device=dev)
    x = torch.randn(1, 3, 2, 8, device=dev, requires_grad=True)
    z = torch.randn(3, 10, device=dev, requires_grad=True)
    cos, sin = A.rope_tables(3, 8, device=dev)

    def pack(tensor):
        raise KeyError("packed")

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda tensor: tensor):
        for call in (lambda: A.embedding(w, t), lambda: A.qk_norm_rope(x, x, cos, sin), lambda: A.cross_entropy(z, t)):
            with pytest.raises(KeyError, match="packed"):
                call()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(dev).total_memory
    # the allocator's own limit, a little above what is in use: nothing is asked of the device
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved(dev) + (64 << 20)) / total, dev)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            A.embedding(w.detach(), t[:1].expand(1 << 24))
        with pytest.raises(torch.OutOfMemoryError):
            A.embedding_backward(torch.randn(3, 8, device=dev), t, 1 << 24)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, dev)


# ------------------------------------------------------------------------------------------------------------ embedding
def test_embedding_of_the_widest_rows(dev):
    """Rows whose width rounded up to whole lanes is past 2^31."""
    from dion_amd import embedding, embedding_backward

    dim = 2 ** 31 - 1
    row = torch.randn(1, dim, device=dev, dtype=BF)
    token = torch.zeros(1, dtype=torch.long, device=dev)
    assert torch.equal(embedding(row, token), row)
    assert torch.equal(embedding_backward(row, token, 1), row)


# ---------------------------------------------------------------------------------------------------------- q / k norms
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim, rotary, interleaved", [(80, 40, False), (90, 44, True), (72, 24, False), (96, 96, True), (128, 128, False)])
def test_qk_norm_rope_gradient_of_infinite_upstream_values(dev, dtype, dim, rotary, interleaved):
    """Infinities and NaN stand where the definition has them, whichever lanes hold the channel."""
    from dion_amd import qk_norm_rope_backward, rope_tables
    from oracle import model_ops as O

    g = _gen(dim)
    q, k = torch.randn(1, dim + 1, 2, dim, generator=g).to(dtype), torch.randn(1, dim + 1, 1, dim, generator=g).to(dtype)
    cos, sin = rope_tables(dim + 1, rotary)
    gain = torch.rand(dim, generator=g) + 0.5
    dy = torch.randn(1, dim + 1, 2, dim, generator=g).to(dtype)
    for channel in range(dim):      # a token each, behind the first, whose angle is zero
        dy[0, channel + 1, 0, channel] = math.inf
    (want, _), _ = O.norm_rope_grad(dy, q, cos, sin, gain, interleaved=interleaved)
    got = qk_norm_rope_backward(*(a.to(dev) for a in (dy, k, q, k, cos, sin)), q_gain=gain.to(dev), interleaved=interleaved)[0].cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and want[0, 1:, 0].isinf().any(-1).sum() > dim // 4
    assert torch.equal(got == math.inf, want == math.inf) and torch.equal(got == -math.inf, want == -math.inf)
    assert got[0, :, 1].isfinite().all()


@pytest.mark.parametrize("vocab", [262143, 262144, 262145])
@pytest.mark.parametrize("count", [100, 3000, 30000])
def test_embedding_backward_of_full_bins(dev, count, vocab):
    """Bins of exactly as many ids as the index has threads, and one more id."""
    g = _gen(count)
    tokens = torch.randint(0, vocab, (count,), generator=g)
    tokens[:6] = torch.tensor([vocab - 1, 0, vocab - 1, vocab - 256, 255, vocab - 1])
    _check_table_gradient(dev, torch.randn(count, 5, generator=g), tokens, vocab, F32, padding_idx=255)


def _grad_on_gpu(grad, tokens, vocab):
    """(gradient, sum of absolute terms, number of terms of a row) in float64, on the GPU"""
    g = grad.double()
    total = torch.zeros(vocab, g.size(1), dtype=torch.float64, device=g.device)
    magnitude, count = torch.zeros_like(total), torch.bincount(tokens, minlength=vocab)
    return total.index_add_(0, tokens, g), magnitude.index_add_(0, tokens, g.abs()), count


def _check_on_gpu(grad, tokens, vocab, dtype):
    from dion_amd import embedding_backward

    got = embedding_backward(grad, tokens, vocab, dtype=dtype)
    want, magnitude, count = _grad_on_gpu(grad, tokens, vocab)
    off = (got.double() - want).abs() - (2.0 ** (-8 if dtype == BF else -24) * want.abs() + 1.01 * (count[:, None] + 2) * EPS * magnitude + 1e-38)
    assert off.max() <= 0, f"{off.max().item():.3e} beyond the bound"
    assert torch.equal(got, embedding_backward(grad, tokens, vocab, dtype=dtype)), "not the same bits twice"


# Entries of a piece are 32 from 4.2 million pairs of token and lane on, 16 from 2.1 million: (tokens, columns) that reach either in
# bf16 (8 columns a lane) and fp32 (4), by the index of few tokens and by that of sorted parts.
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count, dim", [(5001, 2048), (9001, 2049), (20000, 2048), (70001, 512)])
def test_embedding_backward_of_long_pieces(dev, count, dim, dtype):
    g = torch.Generator(dev).manual_seed(count)
    vocab = 5000
    u = torch.rand(count, generator=g, device=dev, dtype=torch.float64)
    i = torch.arange(count, device=dev)
    zipf = (2.7 * ((vocab + 2.7) / 2.7) ** u - 2.7).long().clamp(0, vocab - 1)
    grad = torch.randn(count, dim, generator=g, device=dev, dtype=dtype)
    for tokens in (zipf, i // 97 % vocab, torch.full_like(i, 4321), torch.where(i % 5 == 3, 4321, zipf), torch.where(u < 0.3, 0, zipf)):
        _check_on_gpu(grad, tokens, vocab, dtype)


@pytest.mark.parametrize("dtype, dim", [(BF, 72), (F32, 72), (BF, 16392), (F32, 8196), (BF, 32768), (F32, 16384)])
def test_embedding_backward_around_the_borders_of_pieces(dev, dtype, dim):
    """One id between two others of its bin, its run beginning and ending at every distance from the borders of pieces of 8, 16 and 32
    entries (by the widths), in calls too long for one launch."""
    g = torch.Generator(dev).manual_seed(dim)
    grad = torch.randn(1100, dim, generator=g, device=dev, dtype=dtype)
    for lead in (0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64):
        for run in (1050 - lead, 1023, 33):
            tokens = torch.cat([torch.full((n,), id, device=dev) for n, id in ((lead, 2), (run, 258), (1100 - lead - run, 514))])
            _check_on_gpu(grad, tokens[torch.randperm(1100, generator=g, device=dev)], 600, dtype)


@pytest.mark.parametrize("dtype, gain_dtype", [(BF, F32), (F32, BF), (BF, BF), (F32, F32)])
@pytest.mark.parametrize("case", [(7, 1021, 6, 2, 90, 44, True, True, True), (2, 2051, 32, 8, 128, 128, False, True, True),
                                  (2, 1500, 3, 1, 22, 6, False, True, True), (5, 901, 12, 12, 64, 48, False, True, True)])
def test_qk_norm_rope_gradient_of_many_heads(dev, case, dtype, gain_dtype):
    """More heads than the workgroups of a gradient with gains have lane groups, so that each takes several, and a ragged rest; the
    oracle runs on the GPU, in float64."""
    from dion_amd import qk_norm_rope_backward
    from oracle import model_ops as O

    q, k, cos, sin, options, dy = _qk_problem(dev, case, dtype, gain_dtype)
    grads = qk_norm_rope_backward(*dy, q, k, cos, sin, **options)
    d = q.size(-1)
    for w, (x, name) in enumerate(((q, "q"), (k, "k"))):
        (dx, mx), (dgain, mg) = O.norm_rope_grad(dy[w], x, cos, sin, options[name + "_gain"], options["positions"], 1e-6, options["interleaved"])
        u = 2.0 ** (-8 if dtype == BF else -24)
        off = (grads[w].double() - dx).abs() - (u * dx.abs() + 1.01 * (2 * d + 24) * EPS * mx + 1e-38)
        assert off.max() <= 0, f"d{name}: {off.max().item():.3e} beyond the bound"
        # a term of the gain's gradient (d + 24), and the additions that it passes through: at most 32 heads of a lane group, 8 between the
        # lanes and wavefronts, 32 where the workgroups are joined
        u = 2.0 ** (-8 if gain_dtype == BF else -24)
        off = (grads[2 + w].double() - dgain).abs() - (u * dgain.abs() + 1.01 * (d + 24 + 72) * EPS * mg + 1e-38)
        assert off.max() <= 0, f"gain of {name}: {off.max().item():.3e} beyond the bound"
    for a, b in zip(grads, qk_norm_rope_backward(*dy, q, k, cos, sin, **options)):
        assert torch.equal(a, b), "not the same bits twice"


def test_table_gradient_over_its_own_input_is_refused(dev):
    """A table that lies over the gradient it is made from; one beside it in the same rows is taken."""
    from dion_amd import embedding_backward
    from dion_amd._lib import DionAmdError

    both = torch.randn(600, 24, device=dev)
    tokens = torch.randint(0, 600, (600,), generator=_gen(1)).to(dev)
    grad = both[:, :8].contiguous()
    want = embedding_backward(grad, tokens, 600)
    for out in (grad, grad.view(-1)[:4800].view(600, 8)):
        with pytest.raises(DionAmdError, match="overlap"):
            embedding_backward(grad, tokens, 600, out=out)
    with pytest.raises(DionAmdError, match="overlap"):
        embedding_backward(grad[:500], tokens[:500], 500, out=grad[100:])
    assert torch.equal(embedding_backward(both[:, :8], tokens, 600, out=both[:, 8:16]), want) and torch.equal(both[:, 8:16], want)
