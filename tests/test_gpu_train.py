"""GPU parity of the table-training operators (ai_b200.train) against plain
64-bit implementations, at the sizes and values where they can go wrong.

Tolerances. u = 2^-24 is a float32 rounding's relative size; U[type] the
output type's (2^-24, 2^-8, 2^-11), with its smallest step for values near
zero. A lookup multiplies once and rounds once. A gradient row of c tokens
is c - 1 float32 additions in some order and one product: (c + 1)·u times
the sum of magnitudes. The softmax sums are described at ``_sum_error``.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
TYPES = ["float32", "bfloat16", "float16"]
U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}


def _dt(name):
    import torch

    return getattr(torch, name)


def _name(t):
    return str(t.dtype).replace("torch.", "")


def _gen(cuda, seed):
    import torch

    return torch.Generator(device=cuda).manual_seed(seed)


def _randn(shape, g, cuda, dtype="float32"):
    import torch

    return torch.randn(*shape, generator=g, device=cuda).to(_dt(dtype))


def _near(got, want, err):
    """|got - want| <= err plus the output type's own rounding, NaN and
    infinities in the same places."""
    import torch

    assert got.shape == want.shape, (got.shape, want.shape)
    k = _name(got)
    x, y = got.double(), want.double()
    fine = torch.isfinite(y)
    assert torch.equal(torch.isnan(x), torch.isnan(y))
    off = ~fine & ~torch.isnan(y)
    assert torch.equal(x[off], y[off])
    bound = (err if torch.is_tensor(err) else torch.full_like(y, err)) + U[k] * y.abs() * (1 + 2 * U[k]) + TINY[k]
    d = (x - y).abs()
    ok = ((d <= bound) | ~fine).all()
    assert ok, (float((d - bound)[fine].max()), float(d[fine].max()), (d > bound).nonzero()[:4].tolist())


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("yt", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (5, 7, 3), (33, 100, 768), (129, 50, 769), (7, 9, 256), (1000, 2048, 132)])
def test_lookup(cuda, wt, yt, n, vocab, dim):
    import torch

    from ai_b200 import train

    g = _gen(cuda, n + dim)
    w = _randn((vocab, dim), g, cuda, wt)
    ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int32)
    scale = dim ** 0.5
    y = train.Embedding(w, ids, scale=scale, dtype=_dt(yt))
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    want = w[ids.long()].double() * s32
    _near(y, want, u * want.abs())


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("skip", [0, 1, 2, 4])
def test_lookup_views(cuda, wt, skip):
    """Tables that begin anywhere and whose rows are further apart than their
    length, and a column-major one."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 3)
    whole = _randn((40, 80), g, cuda, wt)
    ids = torch.randint(0, 40, (3, 11), generator=g, device=cuda, dtype=torch.int32)
    for w in (whole[:, skip:skip + 64], whole.t()[skip:, :40]):
        got = train.Embedding(w, ids % w.shape[0])
        assert got.shape == (3, 11, w.shape[1])
        assert torch.equal(got, w[(ids % w.shape[0]).long()])


def test_lookup_padding_and_empty(cuda):
    import torch

    from ai_b200 import train

    w = _randn((6, 20), _gen(cuda, 1), cuda)
    ids = torch.tensor([0, 3, -1, 5], dtype=torch.int32, device=cuda)
    y = train.Embedding(w, ids, padding=-1)
    assert torch.equal(y[[0, 1, 3]], w[[0, 3, 5]]) and not y[2].any()
    ids = torch.tensor([0, 3, 0], dtype=torch.int32, device=cuda)
    y = train.Embedding(w, ids, padding=0)
    assert not y[0].any() and not y[2].any() and torch.equal(y[1], w[3])
    assert train.Embedding(w, ids[:0]).shape == (0, 20)
    train.Check(cuda)


def test_ids_out_of_range_are_reported(cuda):
    """They read and write nothing; the next check names them, once."""
    import torch

    from ai_b200 import _lib, train

    w = _randn((6, 8), _gen(cuda, 1), cuda)
    ids = torch.tensor([1, 6, -2, 2 ** 31 - 1, 5], dtype=torch.int32, device=cuda)
    y = train.Embedding(w, ids)
    with pytest.raises(_lib.FGError) as e:
        train.Check(cuda)
    assert e.value.code == _lib.FG_EINVAL
    assert not y[1:4].any() and torch.equal(y[[0, 4]], w[[1, 5]])
    dy = torch.ones(5, 8, device=cuda)
    for call in (lambda: train.EmbeddingGrad(dy, ids, 6), lambda: train.EmbeddingGradRows(dy, ids, 6),
                 lambda: train.LogProbs(w, ids + 0), lambda: train.LogProbs(w, ids[:1].expand(6) + 7)):
        try:
            call()
        except train.TensorError:  # five targets for six rows
            continue
        with pytest.raises(_lib.FGError):
            train.Check(cuda)
    train.Check(cuda)
    grad = train.EmbeddingGrad(dy, ids, 6)
    assert float(grad.sum()) == 16.0
    with pytest.raises(_lib.FGError):
        train.Check(cuda)


# --------------------------------------------------------------- gradients
def _id_patterns(n, vocab, g, cuda):
    import torch

    arange = torch.arange(n, device=cuda)
    yield "spread", torch.randint(0, vocab, (n,), generator=g, device=cuda)
    yield "one", torch.full((n,), vocab - 1, device=cuda)
    yield "falling", (n - 1 - arange) % vocab
    yield "runs", (arange // 32) % vocab
    frequent = (vocab ** torch.rand(n, generator=g, device=cuda, dtype=torch.float64)).long() - 1
    yield "frequent", frequent.clamp(0, vocab - 1)


def _grad_want(dy, ids, vocab, scale, padding):
    """(sum, error bound) of every row, in 64 bits."""
    import torch

    kept = (ids != padding) & (ids >= 0)
    i = ids.long()[kept]
    d = dy.double()[kept]
    want = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device).index_add_(0, i, d)
    size = torch.zeros_like(want).index_add_(0, i, d.abs())
    many = torch.zeros(vocab, dtype=torch.float64, device=dy.device).index_add_(0, i, torch.ones_like(d[:, 0]))
    return want * scale, (many[:, None] + 1) * u * size * abs(scale) * (1 + 1e-6)


def _check_rows(r, want, err, ids, padding):
    import torch

    kept = ids[(ids != padding) & (ids >= 0)].long()
    met = torch.unique(kept)
    n = len(met)
    assert int(r.Count) == n
    assert torch.equal(r.Ids[:n].long(), met) and bool((r.Ids[n:] == -1).all())
    assert not r.Rows[n:].any()
    _near(r.Rows[:n], want[met], err[met])


@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (2, 3, 5), (31, 7, 64), (32, 32, 33), (33, 1023, 768), (64, 1, 128),
                                         (1000, 1024, 130), (1025, 1025, 40), (4097, 2048, 96), (5000, 300, 769),
                                         (20000, 262144, 64)])
def test_grad(cuda, n, vocab, dim):
    import torch

    from ai_b200 import train

    g = _gen(cuda, n)
    dy = _randn((n, dim), g, cuda)
    for what, ids in _id_patterns(n, vocab, g, cuda):
        ids = ids.int()
        want, err = _grad_want(dy, ids, vocab, 2.0, -1)
        got = train.EmbeddingGrad(dy, ids, vocab, scale=2.0)
        _near(got, want, err)
        assert torch.equal(got, train.EmbeddingGrad(dy, ids, vocab, scale=2.0)), what
        r = train.EmbeddingGradRows(dy, ids, vocab, scale=2.0)
        _check_rows(r, want, err, ids, -1)
    train.Check(cuda)


@pytest.mark.parametrize("yt", TYPES)
@pytest.mark.parametrize("gt", TYPES)
@pytest.mark.parametrize("dim", [128, 65, 768])
def test_grad_types_and_padding(cuda, yt, gt, dim):
    import torch

    from ai_b200 import train

    g = _gen(cuda, 11)
    n, vocab, scale = 700, 90, 0.75
    dy = _randn((n, dim), g, cuda, yt)
    ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int32)
    ids[100:300] = 7
    ids[::5] = 4
    ids[::9] = -1
    for padding in (-1, 4):
        i = torch.where(ids == -1, torch.tensor(padding, dtype=torch.int32, device=cuda), ids)
        want, err = _grad_want(dy, i, vocab, scale, padding)
        got = train.EmbeddingGrad(dy, i, vocab, scale=scale, padding=padding, dtype=_dt(gt))
        assert _name(got) == gt
        _near(got, want, err)
        r = train.EmbeddingGradRows(dy, i, vocab, scale=scale, padding=padding, dtype=_dt(gt))
        _check_rows(r, want, err, i, padding)
        # added to what is there; rows without a token keep their bits
        old = _randn((vocab, dim), g, cuda, gt)
        new = train.EmbeddingGrad(dy, i, vocab, scale=scale, padding=padding, out=old.clone(), accumulate=True)
        sum64 = old.double() + want
        _near(new, sum64, err + u * (want.abs() + sum64.abs()))
        still = want.abs().sum(1) == 0
        assert torch.equal(new[still], old[still]) and (padding != 4 or bool(still[4]))


def test_grad_of_nothing(cuda):
    import torch

    from ai_b200 import train

    dy = torch.ones(50, 12, device=cuda)
    pads = torch.zeros(50, dtype=torch.int32, device=cuda)
    assert not train.EmbeddingGrad(dy, pads, 40, padding=0).any()
    r = train.EmbeddingGradRows(dy, pads, 40, padding=0)
    assert int(r.Count) == 0 and bool((r.Ids == -1).all()) and not r.Rows.any()
    assert not train.EmbeddingGrad(dy[:0], pads[:0], 40).any()
    assert train.EmbeddingGrad(dy[:0], pads[:0], 0).shape == (0, 12)
    r = train.EmbeddingGradRows(dy[:0], pads[:0], 40)
    assert int(r.Count) == 0 and r.Rows.shape == (0, 12) and r.Ids.shape == (0,)
    out = torch.ones(40, 12, device=cuda)
    assert train.EmbeddingGrad(dy[:0], pads[:0], 40, out=out, accumulate=True).eq(1).all()


@pytest.mark.parametrize("yt", TYPES)
def test_grad_views(cuda, yt):
    """Gradients with 3 dimensions, rows apart, an odd start, columns first,
    and an output with rows apart whose gaps stay as they are."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 5)
    whole = _randn((70, 100), g, cuda, yt)
    ids = torch.randint(0, 20, (70,), generator=g, device=cuda, dtype=torch.int32)
    for dy in (whole[:, 1:65], whole[:, 4:36], whole.t().contiguous().t()[:, :31]):
        want, err = _grad_want(dy, ids, 20, 1.0, -1)
        _near(train.EmbeddingGrad(dy, ids, 20), want, err)
        three = dy.reshape(7, 10, -1)
        _near(train.EmbeddingGrad(three, ids.view(7, 10), 20), want, err)
        buf = torch.full((20, dy.shape[1] + 3), 9.0, device=cuda)
        train.EmbeddingGrad(dy, ids, 20, out=buf[:, :dy.shape[1]])
        _near(buf[:, :dy.shape[1]], want, err)
        assert buf[:, dy.shape[1]:].eq(9).all()


def test_grad_wide_keys_and_many_tokens(cuda):
    """Ids of 21 to 31 bits, and more tokens than one group of blocks sorts."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 6)
    n = 300000
    dy = _randn((n, 4), g, cuda)
    for vocab in (1 << 20, (1 << 20) + 3, 2 ** 31 - 2):
        ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int64).int()
        ids[::3] = vocab - 1
        ids[1::7] = 0
        r = train.EmbeddingGradRows(dy, ids, vocab)
        met, at = torch.unique(ids.long(), return_inverse=True)
        want = torch.zeros(len(met), 4, dtype=torch.float64, device=cuda).index_add_(0, at, dy.double())
        size = torch.zeros_like(want).index_add_(0, at, dy.double().abs())
        many = torch.bincount(at).double()
        assert int(r.Count) == len(met) and torch.equal(r.Ids[:len(met)].long(), met)
        _near(r.Rows[:len(met)], want, (many[:, None] + 1) * u * size)
        assert not r.Rows[len(met):].any()


def test_offsets_past_32_bits(cuda):
    """A table and a gradient whose last rows lie past 2^31 values."""
    import torch

    from ai_b200 import train

    vocab, dim = 2_900_000, 768
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device=cuda)
    table[-3:] = 2.0
    ids = torch.tensor([vocab - 1, 5, vocab - 3], dtype=torch.int32, device=cuda)
    y = train.Embedding(table, ids, scale=3.0)
    assert y[[0, 2]].eq(6).all() and not y[1].any()
    dy = torch.ones(3, dim, dtype=torch.bfloat16, device=cuda)
    got = train.EmbeddingGrad(dy, ids, vocab, out=table.fill_(7.0))
    assert got[[vocab - 1, vocab - 3, 5]].eq(1).all()
    assert float(got[-4:].float().sum()) == 2 * dim and float(got[:6].float().sum()) == dim
    assert int(got[: vocab // 2].count_nonzero()) + int(got[vocab // 2:].count_nonzero()) == 3 * dim
    # the same places as token gradients
    ids = torch.full((vocab,), -1, dtype=torch.int32, device=cuda)
    ids[-2:] = 1
    ids[4] = 0
    table.fill_(0)
    table[-2:] = 1.5
    table[4] = 0.25
    got = train.EmbeddingGrad(table, ids, 2, dtype=torch.float32)
    assert got[1].eq(3).all() and got[0].eq(0.25).all()


def test_operators_follow_their_stream(cuda):
    import torch

    from ai_b200 import train

    g = _gen(cuda, 8)
    side = torch.cuda.Stream(cuda)
    dy = _randn((50000, 256), g, cuda)
    ids = torch.randint(0, 5000, (50000,), generator=g, device=cuda, dtype=torch.int32)
    want = train.EmbeddingGrad(dy, ids, 5000)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            late = torch.empty_like(dy).fill_(9.0)  # the operator must wait for what its stream does
            late.copy_(dy)
            got = train.EmbeddingGrad(late, ids, 5000)
            rows = train.EmbeddingGradRows(late, ids, 5000)
            norm = train.ClipGradNorm([got.clone()], 1.0)
    side.synchronize()
    assert torch.equal(got, want)
    n = int(rows.Count)
    assert torch.equal(rows.Rows[:n], want[rows.Ids[:n].long()])
    assert abs(float(norm) - float(want.double().norm())) <= 1e-6 * float(norm)


# ------------------------------------------------------- log probabilities
def _sum_error(width, entropy):
    """Relative error of s1 = Σ e^d. A term's d = (x − m)·scale has two
    roundings and the exponential's argument (a product with log2 e, itself
    rounded) two more, 4u·|d| in all, and the exponential at most 4u of its own; Σ e^d·|d| / s1 is at most the entropy.
    The additions: at most width / 64 + 32 in a row."""
    return u * (4 * entropy + 4 + width / 64 + 32)


def _logprobs_want(x, t, scale):
    import torch

    z = x.double() * scale
    m = z.amax(1, keepdim=True)
    empty = (z == -math.inf).all(1)
    d = z - torch.where(empty[:, None], torch.zeros_like(m), m)
    e = torch.exp(d)
    s1 = e.sum(1)
    s2 = torch.where(e == 0, torch.zeros_like(d), e * d).sum(1)
    logs = torch.log(s1)
    dt = d.gather(1, t.long().clamp(min=0)[:, None])[:, 0]
    logp = torch.where(empty, torch.full_like(logs, -math.inf), dt - logs)
    logp = torch.where(t < 0, torch.zeros_like(logp), logp)
    H = torch.where(empty, torch.zeros_like(logs), logs - s2 / s1)
    lse = m[:, 0] + logs
    lse = torch.where(empty, torch.full_like(logs, -math.inf), lse)
    return d, logs, s2 / s1, logp, H, lse, empty


def _check_logprobs(x, t, scale, top):
    """LogProbs of x against 64 bits; the alternatives against a stable sort."""
    import torch

    from ai_b200 import train

    scale = float(torch.tensor(scale, dtype=torch.float32))
    r = train.LogProbs(x, t, scale=scale, top=top)
    d, logs, mean, logp, H, lse, empty = _logprobs_want(x, t, scale)
    fin = lambda v: torch.where(torch.isfinite(v), v, torch.zeros_like(v))  # noqa: E731
    tol = _sum_error(x.shape[1], fin(H).clamp(min=0)) + u * fin(logs).abs() * 2
    dt = fin(d.gather(1, t.long().clamp(min=0)[:, None])[:, 0])
    _near(r.LogProb, logp, tol + u * (3 * dt.abs() + fin(logp).abs()))
    _near(r.LogSum, lse, tol + u * (fin(lse) - fin(logs)).abs() * 2)
    _near(r.Entropy, H, tol * (2 + 2 * fin(mean).abs()) + 2 * u * fin(mean).abs() + tol * fin(mean).abs())
    if top:
        value, index = x.float().sort(dim=1, descending=True, stable=True)
        assert torch.equal(r.TopIndex.long(), index[:, :top])
        dk = d.gather(1, index[:, :top])
        want = torch.where(empty[:, None], torch.full_like(dk, -math.inf), dk - logs[:, None])
        _near(r.TopLogProb, want, tol[:, None] + u * (3 * fin(dk).abs() + fin(want).abs()))
    else:
        assert r.TopIndex is None and r.TopLogProb is None
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,top", [(1, 1, 1), (3, 2, 2), (5, 31, 7), (4, 33, 33), (7, 64, 64), (2, 257, 20),
                                            (33, 1000, 8), (9, 4097, 64), (300, 513, 3), (2, 30011, 20), (1, 262144, 20),
                                            (1, 100003, 64), (150, 8192, 8), (40, 12288, 1), (3, 70000, 0)])
def test_logprobs(cuda, dtype, rows, width, top):
    import torch

    g = _gen(cuda, width)
    x = _randn((rows, width), g, cuda, dtype) * 3
    t = torch.randint(0, width, (rows,), generator=g, device=cuda, dtype=torch.int32)
    t[rows // 2:rows // 2 + rows // 3] = -1
    _check_logprobs(x, t, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,pad,skip", [(100, 1, 0), (1001, 7, 3), (4096, 8, 0), (4096, 3, 1), (20000, 5, 2)])
def test_logprobs_views(cuda, dtype, width, pad, skip):
    """Rows that begin anywhere, and columns first."""
    import torch

    g = _gen(cuda, width + pad)
    buf = _randn((6, width + pad + skip), g, cuda, dtype)
    t = torch.randint(0, width, (6,), generator=g, device=cuda, dtype=torch.int32)
    _check_logprobs(buf[:, skip:skip + width], t, 10.0, 5)
    if width < 2000:
        _check_logprobs(buf[:, skip:skip + width].t().contiguous().t(), t, 10.0, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [40, 1500, 9000, 66000])
def test_logprobs_orders_and_ties(cuda, dtype, width):
    """Rising and falling rows, equal values, both zeros, few distinct values."""
    import torch

    g = _gen(cuda, width)
    top = min(64, width)
    up = torch.arange(width, device=cuda, dtype=torch.float32) / width
    few = torch.randint(0, 3, (width,), generator=g, device=cuda).float()
    zeros = torch.where(few > 1, torch.tensor(-0.0, device=cuda), torch.tensor(0.0, device=cuda))
    late = torch.zeros(width, device=cuda)
    late[-5:] = 1
    x = torch.stack([up, up.flip(0), torch.full_like(up, 2.5), few, zeros, late, -late]).to(_dt(dtype))
    t = torch.arange(7, device=cuda, dtype=torch.int32)
    _check_logprobs(x, t, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [7, 600, 5000, 40000])
def test_logprobs_masked_and_not_finite(cuda, dtype, width):
    """Masks of -inf and of the type's lowest value, rows with nothing left,
    rows with one entry left, NaN and +inf."""
    import torch

    inf, low = math.inf, torch.finfo(_dt(dtype)).min
    x = _randn((12, width), _gen(cuda, width), cuda, dtype)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = -inf
    x[2, width - 1] = 1.0
    x[3] = low
    x[4, 1:] = low
    x[5, 3] = math.nan
    x[6, 2] = inf
    x[7] = math.nan
    x[8, :width // 2] = -inf
    x[9] = -inf
    x[9, 5] = math.nan
    x[10, :] = inf
    x[11, 1:] = -inf
    t = torch.full((12,), 3, dtype=torch.int32, device=cuda)
    t[2] = width - 1
    t[8] = 0
    r = _check_logprobs(x, t, 1.0, 5)
    assert r.LogProb[1] == -inf and r.Entropy[1] == 0 and r.TopIndex[1].tolist() == [0, 1, 2, 3, 4]
    assert torch.isnan(r.LogProb[5]) and torch.isnan(r.LogSum[6]) and torch.isnan(r.Entropy[7])


def test_logprobs_past_32_bits(cuda):
    import torch

    from ai_b200 import train

    rows, width = 33000, 66000
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda)
    x[-1, 7] = 20.0
    x[-2, width - 1] = 30.0
    t = torch.zeros(rows, dtype=torch.int32, device=cuda)
    t[-1], t[-2] = 7, width - 1
    r = train.LogProbs(x, t, top=1)
    assert r.TopIndex[-2:, 0].tolist() == [width - 1, 7] and not r.TopIndex[:-2].any()
    logp = 20.0 - math.log(math.exp(20.0) + width - 1)
    assert abs(float(r.LogProb[-1]) - logp) <= 2e-3 * abs(logp) + 1e-6
    train.LogProbsGrad(x, t, r.LogSum, torch.ones(rows, device=cuda), out=x)
    p = math.exp(-math.log(width))
    got = x[0].double()
    assert abs(float(got[0]) - (1 - p)) < 2 ** -8 and abs(float(got[1]) + p) < p * 2 ** -8
    last = x[-1].double()
    e = width / math.exp(20.0)
    assert abs(float(last[7]) - e) < 0.05 * e and abs(float(last[6]) + math.exp(-20.0)) < 0.01 * math.exp(-20.0)


def _grad_rows_want(x, t, lse, H, dl, dh, scale):
    """(gradient, error bound): p = e^(z − lse) has the relative error of its
    argument, 4u(|z| + |lse|), the exponential's 4u and the entropy factor's."""
    import torch

    z = x.double() * scale
    lse, dl = lse.double()[:, None], dl.double()[:, None]
    empty = lse == -math.inf
    logp = z - torch.where(empty, torch.zeros_like(lse), lse)
    p = torch.exp(logp)
    rel = 4 * u * (torch.where(p == 0, torch.zeros_like(z), z).abs() + lse.abs()) + 6 * u
    hit = torch.zeros_like(p)
    at = torch.arange(len(t), device=x.device)[t >= 0]
    hit[at, t.long()[t >= 0]] = 1
    dl = torch.where(t[:, None] < 0, torch.zeros_like(dl), dl)
    want = dl * (hit - p)
    err = dl.abs() * (p * rel + 2 * u * (hit + p))
    if dh is not None:
        dh, H = dh.double()[:, None], H.double()[:, None]
        f = torch.where(p == 0, torch.zeros_like(p), logp + H)
        want = want - dh * p * f
        err = err + dh.abs() * p * (f.abs() * (rel + 4 * u) + 2 * u * (torch.where(p == 0, torch.zeros_like(z), z).abs() + lse.abs() + H.abs()))
    zero = torch.zeros_like(want)
    want = torch.where(empty, zero, want * scale)
    err = torch.where(empty, zero, (err + 3 * u * want.abs() / scale) * scale)
    # below the exponential's smallest normal result float32 gives 0
    return want, torch.nan_to_num(err, nan=0.0) + scale * 2.0 ** -125 * (dl.abs().amax() + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,pad", [(1, 1, 0), (3, 5, 0), (17, 33, 1), (4, 1024, 0), (5, 4099, 5), (3, 30011, 0),
                                            (1, 262144, 0), (200, 800, 8)])
@pytest.mark.parametrize("scale,with_entropy", [(1.0, False), (1.0, True), (20.0, True)])
def test_logprobs_grad(cuda, dtype, rows, width, pad, scale, with_entropy):
    import torch

    from ai_b200 import train

    g = _gen(cuda, rows + width)
    buf = _randn((rows, width + pad), g, cuda, dtype) * (3 / scale)
    x = buf[:, :width]
    if rows > 3:
        x[1] = -math.inf
        x[2, ::3] = -math.inf
        x[3] = torch.finfo(_dt(dtype)).min
    t = torch.randint(0, width, (rows,), generator=g, device=cuda, dtype=torch.int32)
    if rows > 1:
        t[0] = -1
    _, _, _, _, H, lse, _ = _logprobs_want(x, t, scale)
    H, lse = H.float(), lse.float()
    dl, dh = torch.randn(rows, generator=g, device=cuda), torch.randn(rows, generator=g, device=cuda)
    dh = dh if with_entropy else None
    want, err = _grad_rows_want(x, t, lse, H, dl, dh, scale)
    kept = buf.clone()
    got = train.LogProbsGrad(x, t, lse, dl, entropy=H, dentropy=dh, scale=scale)
    assert torch.equal(buf.view(torch.uint8) if buf.is_contiguous() else buf, kept.view(torch.uint8)) and _name(got) == dtype
    _near(got, want, err)
    # in place, the values between the rows untouched
    train.LogProbsGrad(x, t, lse, dl, entropy=H, dentropy=dh, scale=scale, out=x)
    assert torch.equal(x, got) and torch.equal(buf[:, width:], kept[:, width:])


def test_logprobs_grad_not_finite(cuda):
    import torch

    from ai_b200 import train

    x = torch.zeros(3, 700, device=cuda)
    x[0, 4] = math.nan
    x[1, 5] = math.inf
    t = torch.zeros(3, dtype=torch.int32, device=cuda)
    r = train.LogProbs(x, t)
    got = train.LogProbsGrad(x, t, r.LogSum, torch.ones(3, device=cuda))
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2]).all()


def test_logprobs_grad_against_differences(cuda):
    """The step of the loss along every logit, from 64-bit losses."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 77)
    rows, width, scale, h = 4, 23, 3.0, 1e-4
    x = _randn((rows, width), g, cuda)
    t = torch.tensor([1, 22, -1, 9], dtype=torch.int32, device=cuda)
    dl, dh = torch.randn(rows, generator=g, device=cuda), torch.randn(rows, generator=g, device=cuda)

    def loss(z):  # [.., rows, width]
        logp = torch.log_softmax(z * scale, -1)
        H = -(logp.exp() * logp).sum(-1)
        picked = logp.gather(-1, t.long().clamp(min=0)[:, None].expand(*z.shape[:-1], 1))[..., 0]
        return (torch.where(t < 0, torch.zeros_like(picked), picked) * dl.double() + H * dh.double()).sum(-1)

    step = h * torch.eye(rows * width, dtype=torch.float64, device=cuda).view(-1, rows, width)
    want = ((loss(x.double() + step) - loss(x.double() - step)) / (2 * h)).view(rows, width)
    r = train.LogProbs(x, t, scale=scale)
    got = train.LogProbsGrad(x, t, r.LogSum, dl, entropy=r.Entropy, dentropy=dh, scale=scale).double()
    # third derivatives of size scale^3 · |weights|: h²·27/6, and float32
    assert float((got - want).abs().max()) <= 27 * h * h * 8 + 64 * u * scale * 8


def test_embedding_grad_against_differences(cuda):
    """The lookup is linear: the loss's difference along a row is its gradient."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 78)
    w, dy = _randn((5, 6), g, cuda), _randn((40, 6), g, cuda)
    ids = torch.randint(0, 5, (40,), generator=g, device=cuda, dtype=torch.int32)
    got = train.EmbeddingGrad(dy, ids, 5, scale=3.0).double()

    def loss(w):
        return float((train.Embedding(w, ids, scale=3.0).double() * dy.double()).sum())

    for v in range(5):
        for c in range(6):
            step = torch.zeros_like(w)
            step[v, c] = 0.5
            diff = loss(w + step) - loss(w - step)
            assert abs(diff - float(got[v, c])) <= 40 * 8 * u * 3 * 4 * 40


# ---------------------------------------------------------------- clipping
def _clip_want(grads, max_norm):
    total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    c = max_norm / total if math.isfinite(total) and total > max_norm else 1.0
    return total, [g.double() * c for g in grads], c


@pytest.mark.parametrize("types", [("float32",), ("bfloat16",), ("float16",), ("float32", "bfloat16", "float16")])
@pytest.mark.parametrize("sizes", [(1,), (3, 0, 5), (768, 768 * 768, 1, 256), (8191, 8192, 8193, 100001), tuple(range(1, 40))])
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clip(cuda, types, sizes, max_norm):
    """In place and apart, in one buffer so that tensors begin anywhere."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, sum(sizes))
    bufs = {k: _randn((sum(sizes) + 1,), g, cuda, k) for k in types}
    grads, at = [], 1
    for i, n in enumerate(sizes):
        grads.append(bufs[types[i % len(types)]][at:at + n])
        at += n
    norm, want, c = _clip_want(grads, max_norm)
    outs = [torch.empty_like(x) for x in grads]
    kept = [x.clone() for x in grads]
    got = train.ClipGradNorm(grads, max_norm, out=outs)
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - norm) <= 4 * u * norm
    for o, w, x, k in zip(outs, want, grads, kept):
        _near(o, w, 4 * u * w.abs())
        assert torch.equal(x, k)
        if c == 1.0:
            assert torch.equal(o, k)
    again = train.ClipGradNorm(grads, max_norm)
    assert float(again) == float(got)
    for x, o in zip(grads, outs):
        assert torch.equal(x, o)


def test_clip_many_tensors(cuda):
    """More tensors than one launch takes."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 2)
    grads = [_randn((1 + i % 70,), g, cuda, TYPES[i % 3]) for i in range(2345)]
    norm, want, _ = _clip_want(grads, 1.5)
    got = train.ClipGradNorm(grads, 1.5)
    assert abs(float(got) - norm) <= 4 * u * norm
    for x, w in zip(grads, want):
        _near(x, w, 4 * u * w.abs())


def test_clip_extremes(cuda):
    """Squares past float32's range, norms that are not finite, zeros, a
    limit of 0 and of infinity."""
    import torch

    from ai_b200 import train

    big = torch.full((1000,), 1e30, device=cuda)
    got = train.ClipGradNorm([big], 1.0)
    assert abs(float(got) / (1e30 * math.sqrt(1000)) - 1) < 4 * u
    assert abs(float(big[0]) * math.sqrt(1000) - 1) < 8 * u
    small = torch.full((1000,), 1e-30, device=cuda)
    assert abs(float(train.ClipGradNorm([small], 1.0)) / (1e-30 * math.sqrt(1000)) - 1) < 4 * u
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.ones(5000, device=cuda)
        x[4321] = bad
        kept = x.clone()
        got = float(train.ClipGradNorm([x], 1.0))
        assert (math.isnan(got) if math.isnan(bad) else got == math.inf)
        assert torch.equal(x.nan_to_num(7.0), kept.nan_to_num(7.0))
    z = torch.zeros(100, device=cuda)
    assert float(train.ClipGradNorm([z], 1.0)) == 0 and not z.any()
    x = torch.ones(100, device=cuda)
    assert float(train.ClipGradNorm([x], math.inf)) == 10 and x.eq(1).all()
    assert float(train.ClipGradNorm([x], 0.0)) == 10 and not x.any()
    assert float(train.ClipGradNorm([x[:0]], 1.0)) == 0


def test_clip_past_32_bits(cuda):
    import torch

    from ai_b200 import train

    x = torch.zeros((1 << 31) + 5, dtype=torch.bfloat16, device=cuda)
    x[-1] = 3.0
    x[1] = 4.0
    assert float(train.ClipGradNorm([x], 1.0)) == 5.0
    assert abs(float(x[-1]) - 0.6) <= 0.6 * 2 ** -8 and abs(float(x[1]) - 0.8) <= 0.8 * 2 ** -8


# ---------------------------------------------------------------- refusals
def test_refusals(cuda):
    import torch

    from ai_b200 import train

    x = torch.zeros(4, 8, device=cuda)
    i = torch.zeros(4, dtype=torch.int32, device=cuda)
    f = torch.zeros(4, device=cuda)
    bad = [
        lambda: train.Embedding(x.double(), i),
        lambda: train.Embedding(x[0], i),
        lambda: train.Embedding(x, i.long()),
        lambda: train.Embedding(x, i.cpu()),
        lambda: train.Embedding(x, i, dtype=torch.float64),
        lambda: train.EmbeddingGrad(x, i[:3], 5),
        lambda: train.EmbeddingGrad(x, i, -1),
        lambda: train.EmbeddingGrad(x, i, 5, accumulate=True),
        lambda: train.EmbeddingGrad(x, i, 5, out=torch.zeros(4, 8, device=cuda)),
        lambda: train.EmbeddingGrad(x, i, 5, out=torch.zeros(8, 5, device=cuda).t()),
        lambda: train.EmbeddingGrad(x, i, 5, dtype=torch.float16, out=torch.zeros(5, 8, device=cuda)),
        lambda: train.EmbeddingGradRows(x, i.long(), 5),
        lambda: train.LogProbs(x, i, top=9),
        lambda: train.LogProbs(x, i, top=-1),
        lambda: train.LogProbs(torch.zeros(4, 100, device=cuda), i, top=65),
        lambda: train.LogProbs(x, i, scale=0.0),
        lambda: train.LogProbs(x, i[:2]),
        lambda: train.LogProbs(x[:, :0], i),
        lambda: train.LogProbsGrad(x, i, f[:3], f),
        lambda: train.LogProbsGrad(x, i, f, f, dentropy=f),
        lambda: train.LogProbsGrad(x, i, f, f.double()),
        lambda: train.LogProbsGrad(x, i, f, f, out=x.half()),
        lambda: train.ClipGradNorm([x.t()], 1.0),
        lambda: train.ClipGradNorm([x, x.cpu()], 1.0),
        lambda: train.ClipGradNorm([x], 1.0, out=[]),
        lambda: train.ClipGradNorm([x], math.nan),
        lambda: train.ClipGradNorm([i], 1.0),
    ]
    for call in bad:
        with pytest.raises(train.TensorError):
            call()


# ------------------------------------------- every way the work is divided
@pytest.mark.parametrize("n,vocab,dim", [(40000, 3, 8), (100000, 2, 4), (70000, 1000, 40), (270000, 1000, 12), (265000, 30000, 5)])
def test_grad_long_runs(cuda, n, vocab, dim):
    """Runs of thousands of chunks, more tokens than one cluster sorts, and
    the rows no token met among them."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, n)
    dy = _randn((n, dim), g, cuda)
    ids = torch.randint(0, max(1, vocab - 1), (n,), generator=g, device=cuda, dtype=torch.int32)
    ids[n // 3:2 * n // 3] = 1
    want, err = _grad_want(dy, ids, vocab, 1.0, -1)
    got = train.EmbeddingGrad(dy, ids, vocab)
    _near(got, want, err)
    assert torch.equal(got, train.EmbeddingGrad(dy, ids, vocab))
    _check_rows(train.EmbeddingGradRows(dy, ids, vocab), want, err, ids, -1)
    old = torch.ones(vocab, dim, device=cuda)
    new = train.EmbeddingGrad(dy, ids, vocab, out=old.clone(), accumulate=True)
    _near(new, want + 1, err + u * (want.abs() + (want + 1).abs()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5000, 20001])
def test_grad_of_a_large_table(cuda, dtype, n):
    """Zeros written beside the sort: 262144 rows, few of them met."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, n)
    vocab, dim = 262144, 96
    dy = _randn((n, dim), g, cuda, dtype)
    ids = (vocab ** torch.rand(n, generator=g, device=cuda, dtype=torch.float64)).int().clamp(0, vocab - 1)
    ids[::50] = vocab - 1
    ids[::77] = -1
    want, err = _grad_want(dy, ids, vocab, 0.5, -1)
    out = torch.full((vocab, dim), 3.0, device=cuda, dtype=_dt(dtype))
    got = train.EmbeddingGrad(dy, ids, vocab, scale=0.5, out=out)
    _near(got, want, err)
    still = want.abs().sum(1) == 0
    assert not got[still].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,width,top", [(4000, 1537, 9), (2000, 1100, 33), (900, 2100, 5), (450, 4200, 64), (240, 9000, 20),
                                            (100, 40000, 20), (40, 100001, 64), (9000, 30, 30), (5000, 513, 0)])
def test_logprobs_divisions(cuda, dtype, rows, width, top):
    """One to sixteen warps a row, one to sixteen blocks."""
    import torch

    g = _gen(cuda, rows)
    x = _randn((rows, width), g, cuda, dtype) * 2
    t = torch.randint(-1, width, (rows,), generator=g, device=cuda, dtype=torch.int32)
    _check_logprobs(x, t, 3.0, top)


def test_operators_in_a_graph(cuda):
    """Captured once, replayed on new contents of the same tensors."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 4)
    table = _randn((3000, 128), g, cuda)
    ids = torch.randint(0, 3000, (6000,), generator=g, device=cuda, dtype=torch.int32)
    logits = _randn((64, 5000), g, cuda)
    t = torch.randint(0, 5000, (64,), generator=g, device=cuda, dtype=torch.int32)
    one = torch.ones(64, device=cuda)

    def all_of_them():
        y = train.Embedding(table, ids, scale=2.0)
        dense = train.EmbeddingGrad(y, ids, 3000)
        rows = train.EmbeddingGradRows(y, ids, 3000)
        p = train.LogProbs(logits, t, top=5)
        d = train.LogProbsGrad(logits, t, p.LogSum, one)
        norm = train.ClipGradNorm([dense, rows.Rows, d], 1.0)
        return [y, dense, *rows, *p, d, norm]

    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        all_of_them()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = all_of_them()
    for _ in range(2):
        ids.copy_(torch.randint(0, 3000, (6000,), generator=g, device=cuda, dtype=torch.int32))
        logits.copy_(_randn((64, 5000), g, cuda))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, all_of_them()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n", [7, 1000, 2048, 2049, 5000, 20000])
@pytest.mark.parametrize("vocab", [1 << 10, (1 << 20) + 3, 2 ** 31 - 2])
def test_grad_rows_of_wide_keys(cuda, n, vocab):
    """One to four passes of the sorts that few tokens take."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, n)
    dy = _randn((n, 3), g, cuda)
    ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int64)
    ids[::3], ids[1::5], ids[2::5] = vocab - 1, 0, -1
    r = train.EmbeddingGradRows(dy, ids.int(), vocab)
    keep = ids >= 0
    met, at = torch.unique(ids[keep], return_inverse=True)
    d = dy.double()[keep]
    want = torch.zeros(len(met), 3, dtype=torch.float64, device=cuda).index_add_(0, at, d)
    size = torch.zeros_like(want).index_add_(0, at, d.abs())
    assert int(r.Count) == len(met) and torch.equal(r.Ids[:len(met)].long(), met)
    assert bool((r.Ids[len(met):] == -1).all()) and not r.Rows[len(met):].any()
    _near(r.Rows[:len(met)], want, (torch.bincount(at).double()[:, None] + 1) * u * size)


def test_lookup_of_an_empty_table(cuda):
    import torch

    from ai_b200 import _lib, train

    y = train.Embedding(torch.empty(0, 5, device=cuda), torch.tensor([-1, -1], dtype=torch.int32, device=cuda))
    assert y.shape == (2, 5) and not y.any()
    train.Check(cuda)
    train.Embedding(torch.empty(0, 5, device=cuda), torch.tensor([0], dtype=torch.int32, device=cuda))
    with pytest.raises(_lib.FGError):
        train.Check(cuda)


@pytest.mark.parametrize("n,vocab,dim", [(1024, 700, 301), (1025, 700, 301), (2048, 900, 1023), (1500, 3, 517),
                                         (2048, 50, 2048), (2047, 5000, 385), (1, 70, 33000), (300, 40, 4097)])
def test_grad_of_few_tokens_with_many_columns(cuda, n, vocab, dim):
    import torch

    from ai_b200 import train

    g = _gen(cuda, n + dim)
    dy = _randn((n, dim), g, cuda)
    for what, ids in _id_patterns(n, vocab, g, cuda):
        ids = ids.int()
        want, err = _grad_want(dy, ids, vocab, 0.5, 2)
        got = train.EmbeddingGrad(dy, ids, vocab, scale=0.5, padding=2)
        _near(got, want, err)
        assert torch.equal(got, train.EmbeddingGrad(dy, ids, vocab, scale=0.5, padding=2)), what
        _check_rows(train.EmbeddingGradRows(dy, ids, vocab, scale=0.5, padding=2), want, err, ids, 2)
    train.Check(cuda)


@pytest.mark.parametrize("gt", TYPES)
@pytest.mark.parametrize("n", [3, 900, 2500])
@pytest.mark.parametrize("dim", [1, 3, 7, 33, 130])
def test_grad_zeros_between_rows_met(cuda, gt, n, dim):
    """Zeros for rows in groups of any length, from any start of an output
    with and without gaps between its rows; nothing outside it is written."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, n + dim)
    vocab = 203
    dy = _randn((n, dim), g, cuda)
    ids = torch.randint(0, 12, (n,), generator=g, device=cuda, dtype=torch.int32)
    ids = torch.where(ids < 9, ids * 13 + 30, ids + 60)
    want, err = _grad_want(dy, ids, vocab, 1.0, -1)
    for start, gap in ((0, 0), (1, 0), (5, 0), (3, 2)):
        buf = torch.full((start + vocab * (dim + gap) + 19,), 9.0, dtype=_dt(gt), device=cuda)
        out = buf[start:start + vocab * (dim + gap)].view(vocab, dim + gap)[:, :dim]
        _near(train.EmbeddingGrad(dy, ids, vocab, out=out), want, err)
        out.fill_(9.0)
        assert buf.eq(9).all()


# ------------------------------------------------- forward and gradient together
def _pair_want(x, t, dl, dh, scale):
    """(gradient, error bound) of logprob·dl + H·dh in 64 bits from the logits
    alone. The operators' log p is scale·(x − peak) (two roundings) less log s1
    (``_sum_error``, its own rounding), their H within ``_check_logprobs``'s."""
    import torch

    d, logs, mean, _, H, _, empty = _logprobs_want(x, t, scale)
    fin = lambda v: torch.where(torch.isfinite(v), v, torch.zeros_like(v))  # noqa: E731
    sums = _sum_error(x.shape[1], fin(H).clamp(min=0)) + 2 * u * fin(logs).abs()
    H_err = sums * (2 + 3 * fin(mean).abs()) + 2 * u * fin(mean).abs()
    logp = d - logs[:, None]
    p = torch.exp(logp)
    here = p != 0
    lp_err = torch.where(here, u * (3 * d.abs() + fin(logs).abs()[:, None] + logp.abs()), torch.zeros_like(p)) + sums[:, None]
    rel = lp_err + u * torch.where(here, logp.abs(), torch.zeros_like(p)) * 2 + 6 * u
    hit = torch.zeros_like(p)
    at = torch.arange(len(t), device=x.device)[t >= 0]
    hit[at, t.long()[t >= 0]] = 1
    dl = torch.where(t < 0, torch.zeros_like(dl), dl).double()[:, None]
    want, err = dl * (hit - p), dl.abs() * (p * rel + 2 * u * (hit + p))
    if dh is not None:
        dh = dh.double()[:, None]
        f = torch.where(here, logp + H[:, None], torch.zeros_like(p))
        want = want - dh * p * f
        err = err + dh.abs() * p * (f.abs() * (rel + 4 * u) + lp_err + H_err[:, None])
    zero = torch.zeros_like(want)
    want = torch.where(empty[:, None], zero, want * scale)
    err = torch.where(empty[:, None], zero, (err + 3 * u * want.abs() / scale) * scale)
    # below the exponential's smallest normal result float32 gives 0
    weights = dl.abs().amax() + (0 if dh is None else dh.abs().amax() * 128)
    return want, err + scale * 2.0 ** -125 * (weights + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,pad", [(1, 0), (7, 0), (1000, 0), (1001, 3), (40000, 0)])
@pytest.mark.parametrize("scale", [1.0, 20.0])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_logprobs_pair_of_rows_far_from_zero(cuda, dtype, width, pad, scale, with_entropy):
    """Rows of the type's lowest value, of one large value, with an offset that
    leaves lse no room for log s1, beside ordinary and masked ones: the
    gradient through Peak against 64 bits, from the logits alone."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, width + int(scale))
    far = 3e4 if dtype == "float16" else 1e6
    buf = _randn((9, width + pad), g, cuda, "float32") * (3 / scale)
    buf[0] = torch.finfo(_dt(dtype)).min
    buf[1] = -6e4 if dtype == "float16" else -1e9
    buf[2] += far
    buf[3] -= far
    buf[4] = -math.inf
    buf[5, ::2] = torch.finfo(_dt(dtype)).min
    buf[6, : width // 2] = -math.inf
    buf[7] = torch.finfo(_dt(dtype)).max
    buf = buf.to(_dt(dtype))
    x = buf[:, :width]
    t = torch.randint(0, width, (9,), generator=g, device=cuda, dtype=torch.int32)
    t[8] = -1
    dl = torch.randn(9, generator=g, device=cuda)
    dh = torch.randn(9, generator=g, device=cuda) if with_entropy else None
    want, err = _pair_want(x, t, dl, dh, scale)
    r = train.LogProbs(x, t, scale=scale)
    assert r.Peak.shape == (2, 9) and torch.equal(r.Peak[0], x.float().amax(1))
    kept = buf.clone()
    got = train.LogProbsGrad(x, t, None, dl, entropy=r.Entropy, dentropy=dh, scale=scale, peak=r.Peak)
    _near(got, want, err)
    again = train.LogProbsGrad(x, t, r.LogSum, dl, entropy=r.Entropy, dentropy=dh, scale=scale, peak=r.Peak, out=x)
    assert torch.equal(again, got) and torch.equal(buf[:, width:], kept[:, width:])


def test_logprobs_pair_not_finite(cuda):
    """NaN and +inf reach the gradient through Peak as through LogSum."""
    import torch

    from ai_b200 import train

    x = torch.zeros(4, 700, device=cuda)
    x[0, 4] = math.nan
    x[1, 5] = math.inf
    x[3] = -math.inf
    t = torch.zeros(4, dtype=torch.int32, device=cuda)
    r = train.LogProbs(x, t, top=3)
    assert r.Peak[0, 1] == math.inf and torch.isnan(r.Peak[:, 0]).all() and r.Peak[:, 3].eq(-math.inf).all()
    assert float(r.Peak[1, 2]) == float(r.TopLogProb[2, 0]) == float(r.LogProb[2])
    got = train.LogProbsGrad(x, t, None, torch.ones(4, device=cuda), peak=r.Peak)
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2]).all() and not got[3].any()
    for bad in (r.Peak[0], r.Peak.double(), r.Peak.cpu()):
        with pytest.raises(train.TensorError):
            train.LogProbsGrad(x, t, r.LogSum, torch.ones(4, device=cuda), peak=bad)
    with pytest.raises(train.TensorError):
        train.LogProbsGrad(x, t, None, torch.ones(4, device=cuda))


# --------------------------------------------- what an id out of range touches
def _bad_id(cuda):
    import torch

    from ai_b200 import train

    train.Embedding(torch.ones(6, 8, device=cuda), torch.tensor([9], dtype=torch.int32, device=cuda))


def _check_reports_once(cuda):
    from ai_b200 import _lib, train

    with pytest.raises(_lib.FGError) as e:
        train.Check(cuda)
    assert e.value.code == _lib.FG_EINVAL
    train.Check(cuda)


def test_bad_id_leaves_other_calls_alone(cuda):
    """KMeans and a model's forward with good inputs succeed after it, and the
    report is still there for Check."""
    import torch

    from ai_b200 import cluster, gemma
    from ai_b200 import synthetic as S

    x = _randn((300, 16), _gen(cuda, 9), cuda)
    _bad_id(cuda)
    cluster.KMeans(x, 3, 4, 1)
    _check_reports_once(cuda)
    cfg = S.small_config(layers=1, vocab=256)
    model = gemma.from_synthetic(cfg, S.make_weights(cfg, seed=0), device=0, max_batch_tokens=256)
    try:
        ids, lengths = S.make_ids(2, 16, 1, cfg["vocab_size"]), torch.full((2,), 16, dtype=torch.int32).numpy()
        _bad_id(cuda)
        model.embed_padded(ids, lengths)
        model.check()
        _check_reports_once(cuda)
    finally:
        model.close()


@pytest.mark.parametrize("noalloc", [False, True])
def test_bad_id_does_not_hide_a_wait_that_gave_up(cuda, noalloc):
    """A bad id, then a product whose waits run out under a limit of 1 us: the
    timeout is reported first, then the id."""
    import torch

    from ai_b200 import _lib

    lib = _lib.lib()
    fn = lib.fg_matmul_noalloc if noalloc else lib.fg_matmul
    g = _gen(cuda, 5)
    m, n, k = 512, 512, 8192
    a, w, out = _randn((m, k), g, cuda), _randn((n, k), g, cuda), torch.empty(m, n, device=cuda)

    def product():
        _lib.check(fn(m, n, k, a.data_ptr(), k, w.data_ptr(), k, 1, out.data_ptr(), n, None, _lib.PREC_TF32,
                      torch.cuda.current_stream().cuda_stream))

    product()  # set-up before the limit changes
    _lib.check(lib.fg_synchronize(0))
    try:
        _bad_id(cuda)
        _lib.check(lib.fg_set_wait_limit(0, 1000))
        product()
        rc = lib.fg_synchronize(0)
    finally:
        _lib.check(lib.fg_set_wait_limit(0, 0))
    assert rc == _lib.FG_ETIMEOUT
    _check_reports_once(cuda)


def test_logprobs_results_lie_apart(cuda):
    """Peak and the three sums share an allocation and nothing else."""
    import torch

    from ai_b200 import train

    for rows in (0, 1, 5, 1000):
        x = _randn((rows, 9), _gen(cuda, rows), cuda)
        r = train.LogProbs(x, torch.zeros(rows, dtype=torch.int32, device=cuda))
        parts = [r.LogProb, r.Entropy, r.LogSum, r.Peak[0], r.Peak[1]]
        assert r.Peak.shape == (2, rows) and r.Peak.is_contiguous() and all(p.is_contiguous() and p.shape == (rows,) for p in parts)
        at = sorted((p.data_ptr(), p.data_ptr() + 4 * rows) for p in parts)
        assert rows == 0 or all(a[1] <= b[0] for a, b in zip(at, at[1:]))
        assert torch.equal(r.Peak[0], x.amax(1)) if rows else True
        want = x.double().logsumexp(1) if rows else x.double().sum(1)
        assert torch.allclose(r.LogSum.double(), want, rtol=1e-5, atol=1e-6)


# ------------------------------------------------ norms at the ends of the range
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("value,count,max_norm", [
    (1e38, 1000, 1.0),       # a norm of 3.2e39: inf as a float32
    (3e38, 2, 1e-3),         # 4.2e38
    (1.6e38, 4, 1e-3),       # 3.2e38: finite, the factor 3e-42
    (1.6e38, 4, 1e-30),      # the factor 3e-69
    (2.0 ** 126, 16, 2.0 ** -20),
    (1e37, 30011, 7.0),
    (1e20, 70000, 1e-25),
])
def test_clip_of_the_largest_norms(cuda, dtype, value, count, max_norm):
    """A norm that is not finite as returned changes nothing; a finite one
    clips within one rounding however small the factor."""
    import torch

    from ai_b200 import train

    x = torch.full((count,), value, device=cuda).to(_dt(dtype))
    x[::3] *= -0.5
    kept = x.clone()
    norm = math.sqrt(float((x.double() ** 2).sum()))
    as_float = float(torch.tensor(norm, dtype=torch.float64).float())
    out = torch.empty_like(x)
    got = float(train.ClipGradNorm([x], max_norm, out=[out]))
    assert torch.equal(x, kept)
    assert float(train.ClipGradNorm([x], max_norm)) == got
    assert torch.equal(x, out)
    if math.isinf(as_float):
        assert got == math.inf and torch.equal(x, kept)
        return
    assert abs(got / norm - 1) <= 4 * u
    m32 = float(torch.tensor(max_norm, dtype=torch.float32))
    want = kept.double() * (m32 / norm)
    _near(x, want, 4 * u * want.abs())


# ----------------------------------------------- scales at the ends of the range
def _fits(v, dtype="float32"):
    """64-bit values as the type has them at its ends: infinite past them."""
    import torch

    return torch.where(torch.isinf(v.to(_dt(dtype))), torch.sign(v) * math.inf, v)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width,top", [(8, 0), (9, 5), (3000, 20), (70000, 3)])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 2e-37, 1e-30, 0.5, 1e30, 2e38])
def test_logprobs_of_any_scale(cuda, dtype, width, top, scale):
    """Masked entries have no probability at any scale, and differences past
    float32's range count by what the scale makes of them."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, width)
    most = float(torch.finfo(_dt(dtype)).max)
    near = max(min(1 / scale, most / 8), 1e-30)
    x = _randn((5, width), g, cuda, "float32") * near
    x[1, ::2] = -math.inf
    x[2] = torch.where(x[2] > 0, 0.9 * most, -0.9 * most)
    x[3, ::2] = -most
    x[4] = -math.inf
    x = x.to(_dt(dtype))
    t = torch.randint(0, width, (5,), generator=g, device=cuda, dtype=torch.int32)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    r = train.LogProbs(x, t, scale=scale, top=top)
    d, logs, mean, logp, H, lse, empty = _logprobs_want(x, t, s32)
    fin = lambda v: torch.where(torch.isfinite(v), v, torch.zeros_like(v))  # noqa: E731
    tol = _sum_error(width, fin(H).clamp(min=0)) + u * fin(logs).abs() * 2
    dt = fin(d.gather(1, t.long()[:, None])[:, 0])
    _near(r.LogProb, _fits(logp), tol + u * (3 * dt.abs() + fin(logp).abs()))
    _near(r.LogSum, _fits(lse), tol + u * (fin(lse) - fin(logs)).abs() * 2)
    _near(r.Entropy, H, tol * (2 + 3 * fin(mean).abs()) + 2 * u * fin(mean).abs())
    if top:
        _, index = x.float().sort(dim=1, descending=True, stable=True)
        assert torch.equal(r.TopIndex.long(), index[:, :top])
        dk = d.gather(1, index[:, :top])
        want = torch.where(empty[:, None], torch.full_like(dk, -math.inf), dk - logs[:, None])
        _near(r.TopLogProb, _fits(want), tol[:, None] + u * (3 * fin(dk).abs() + fin(want).abs()))
    if scale > 1e-40:  # a gradient of that scale is below float32's numbers
        dl, dh = torch.randn(5, generator=g, device=cuda), torch.randn(5, generator=g, device=cuda)
        want, err = _pair_want(x, t, dl, dh, s32)
        got = train.LogProbsGrad(x, t, None, dl, entropy=r.Entropy, dentropy=dh, scale=scale, peak=r.Peak)
        _near(got, _fits(want, dtype), err + 2.0 ** -149)


def test_logprobs_refuses_a_scale_too_large(cuda):
    import torch

    from ai_b200 import train

    x, t = torch.zeros(2, 4, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    with pytest.raises(train.TensorError):
        train.LogProbs(x, t, scale=3e38)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clip_of_a_padded_gradient(cuda, dtype, max_norm):
    """The gradient of padded logits has their layout; it clips as a packed one
    does, alone and among others, and what lies between its rows stays."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 21)
    x = _randn((30, 107), g, cuda, dtype)[:, :100]
    t = torch.randint(0, 100, (30,), generator=g, device=cuda, dtype=torch.int32)
    r = train.LogProbs(x, t)
    d = train.LogProbsGrad(x, t, r.LogSum, torch.ones(30, device=cuda))
    assert not d.is_contiguous()
    buf = torch.full((30, 107), 9.0, device=cuda, dtype=_dt(dtype))
    rows = buf[:, :100]
    rows.copy_(d)
    other = _randn((50,), g, cuda)
    for with_other in (False, True):
        def among(a, b):
            return [b, a] if with_other else [a]

        rows.copy_(d)
        packed, b1, b2, b3 = d.contiguous(), other.clone(), other.clone(), other.clone()
        want = float(train.ClipGradNorm(among(packed, b1), max_norm))
        out = among(torch.empty_like(packed), torch.empty_like(b2))
        assert float(train.ClipGradNorm(among(rows, b2), max_norm, out=out)) == want
        assert torch.equal(rows, d) and torch.equal(b2, other)
        assert all(torch.equal(a, b) for a, b in zip(out, among(packed, b1)))
        assert float(train.ClipGradNorm(among(rows, b3), max_norm)) == want
        assert torch.equal(rows, packed) and torch.equal(b3, b1) and buf[:, 100:].eq(9).all()
    with pytest.raises(train.TensorError):
        train.ClipGradNorm([d.t()], 1.0)
    with pytest.raises(train.TensorError):
        train.ClipGradNorm([d.contiguous()], 1.0, out=[rows])


@pytest.mark.parametrize("padding", [2 ** 31, 2 ** 32, -2 ** 31 - 1, 2 ** 40 + 3])
def test_a_padding_that_is_no_id_is_refused(cuda, padding):
    """A padding past int32 named another id's rows by its lower bits."""
    import torch

    from ai_b200 import train

    x, i = torch.ones(4, 8, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    for call in (lambda: train.Embedding(x, i, padding=padding), lambda: train.EmbeddingGrad(x, i, 4, padding=padding),
                 lambda: train.EmbeddingGradRows(x, i, 4, padding=padding)):
        with pytest.raises(train.TensorError):
            call()
    for padding in (2 ** 31 - 1, -2 ** 31):
        assert train.Embedding(x, i, padding=padding).eq(1).all()


# ------------------------------------------- reports, captures, streams, long sums
@pytest.mark.parametrize("n,vocab,dim", [(600, 50, 16), (5000, 300, 33), (20000, 262144, 96), (300000, 1000, 4)])
def test_gradients_skip_and_report_ids_out_of_range(cuda, n, vocab, dim):
    """One launch, a cluster's sort, zeros beside it, tiles through memory: ids
    past the table and negative ones leave no trace but the report."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, n)
    dy = _randn((n, dim), g, cuda)
    ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int32)
    ids[::7], ids[1::11], ids[2::13], ids[3::17] = vocab, -1, -2 ** 31, 2 ** 31 - 1
    good = (ids >= 0) & (ids < vocab)
    kept = torch.where(good, ids, torch.full_like(ids, -5))
    want, err = _grad_want(dy, kept, vocab, 1.0, -5)
    got = train.EmbeddingGrad(dy, ids, vocab, padding=-5)
    _check_reports_once(cuda)
    _near(got, want, err)
    r = train.EmbeddingGradRows(dy, ids, vocab, padding=-5)
    _check_reports_once(cuda)
    _check_rows(r, want, err, kept, -5)
    old = torch.ones(vocab, dim, device=cuda)
    new = train.EmbeddingGrad(dy, ids, vocab, padding=-5, out=old.clone(), accumulate=True)
    _check_reports_once(cuda)
    _near(new, want + 1, err + u * (want.abs() + (want + 1).abs()))


@pytest.mark.parametrize("width,rows", [(9, 4), (700, 3), (70000, 2)])
def test_targets_out_of_range_are_reported(cuda, width, rows):
    """A target past the row counts as none, forward and back."""
    import torch

    from ai_b200 import train

    x = _randn((rows, width), _gen(cuda, width), cuda)
    good = torch.full((rows,), -1, dtype=torch.int32, device=cuda)
    one = torch.ones(rows, device=cuda)
    want = train.LogProbs(x, good)
    dwant = train.LogProbsGrad(x, good, want.LogSum, one, entropy=want.Entropy, dentropy=one)
    dpeak = train.LogProbsGrad(x, good, None, one, entropy=want.Entropy, dentropy=one, peak=want.Peak)
    train.Check(cuda)
    for bad in (width, 2 ** 31 - 1):
        t = good.clone()
        t[-1] = bad
        got = train.LogProbs(x, t)
        _check_reports_once(cuda)
        assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3])) and not got.LogProb.any()
        d = train.LogProbsGrad(x, t, want.LogSum, one, entropy=want.Entropy, dentropy=one)
        _check_reports_once(cuda)
        assert torch.equal(d, dwant)
        d = train.LogProbsGrad(x, t, None, one, entropy=want.Entropy, dentropy=one, peak=want.Peak)
        _check_reports_once(cuda)
        assert torch.equal(d, dpeak)


def test_large_table_gradient_in_a_graph(cuda):
    """The zeros that are written beside the sort, the marks before both and the
    tiled sort, captured once and replayed on new ids."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 14)
    vocab, dim, n, many = 262144, 96, 20000, 270000
    dy, dy2 = _randn((n, dim), g, cuda), _randn((many, 4), g, cuda)
    ids = torch.randint(0, vocab, (n,), generator=g, device=cuda, dtype=torch.int32)
    ids2 = torch.randint(0, 5000, (many,), generator=g, device=cuda, dtype=torch.int32)

    def both():
        return [train.EmbeddingGrad(dy, ids, vocab, scale=0.5), train.EmbeddingGrad(dy2, ids2, 5000),
                *train.EmbeddingGradRows(dy2, ids2, 5000)]

    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = both()
    for low in (1, 100, vocab // 2):
        ids.copy_(torch.randint(0, low, (n,), generator=g, device=cuda, dtype=torch.int32))
        ids2.copy_(torch.randint(0, min(low, 5000), (many,), generator=g, device=cuda, dtype=torch.int32))
        for o in outs:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want, err = _grad_want(dy, ids, vocab, 0.5, -1)
        _near(outs[0], want, err)
        for a, b in zip([o.clone() for o in outs], both()):
            assert torch.equal(a, b)


def test_operators_on_two_streams_at_once(cuda):
    """Calls in flight together share the pool that their scratch comes from,
    and no part of it."""
    import torch

    from ai_b200 import train

    g = _gen(cuda, 15)
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    data = []
    for n, vocab, dim in ((60000, 262144, 64), (280000, 3000, 24)):
        dy = _randn((n, dim), g, cuda)
        ids = (vocab ** torch.rand(n, generator=g, device=cuda, dtype=torch.float64)).int().clamp(0, vocab - 1)
        data.append((dy, ids, vocab, train.EmbeddingGrad(dy, ids, vocab), train.EmbeddingGradRows(dy, ids, vocab),
                     train.ClipGradNorm([dy.clone()], 1.0)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            dy, ids, vocab = data[i][:3]
            with torch.cuda.stream(s):
                got[i].append((train.EmbeddingGrad(dy, ids, vocab), train.EmbeddingGradRows(dy, ids, vocab),
                               train.ClipGradNorm([dy], math.inf)))
    torch.cuda.synchronize()
    for i in range(2):
        for dense, rows, norm in got[i]:
            assert torch.equal(dense, data[i][3]) and torch.equal(norm, data[i][5])
            assert all(torch.equal(a, b) for a, b in zip(rows, data[i][4]))


def _tight(width, H, logs):
    """What the kernel's sums may be off by, relative: a term's exponent 4u·|d|
    and its exponential 4u as in ``_sum_error``; 8 additions and one in a tile,
    the tiles' compensated sum 3, the lanes 5, warps and blocks of a row 10; a
    lane's running maximum moves at most 8 times (a term's own rounding 2u, the
    factor's exponential 4u and two products)."""
    return u * (4 * H + 4 + 9 + 3 + 5 + 10 + 8 * 8) + 2 * u * abs(logs)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(1, 262144), (40, 262144), (3400, 30011)])
def test_logprobs_long_sums(cuda, dtype, rows, width):
    import torch

    from ai_b200 import train

    x = _randn((rows, width), _gen(cuda, rows), cuda, dtype)
    r = train.LogProbs(x, torch.zeros(rows, dtype=torch.int32, device=cuda))
    for i in sorted({0, rows // 2, rows - 1}):
        _, logs, mean, logp, H, lse, _ = _logprobs_want(x[i:i + 1], torch.zeros(1, dtype=torch.int32, device=cuda), 1.0)
        tol = _tight(width, float(H), float(logs))
        assert abs(float(r.LogSum[i]) - float(lse)) <= tol + u * (abs(float(lse)) + 2 * abs(float(lse - logs)))
        assert abs(float(r.LogProb[i]) - float(logp)) <= tol + 2 * u * abs(float(logp))
        assert abs(float(r.Entropy[i]) - float(H)) <= tol * (2 + 3 * abs(float(mean))) + 2 * u * abs(float(mean)) + u * float(H)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logprobs_small_terms_beside_large_ones(cuda, dtype):
    """512 entries of 0, then many whose sum in a tile is below half the last
    bit of a lane's running sum: together 180 of its rounding errors, lost if
    tiles were added without compensation."""
    import torch

    from ai_b200 import train

    rows, width = 3400, 100003
    x = torch.full((rows, width), -16.75, device=cuda, dtype=_dt(dtype))
    x[:, :512] = 0
    r = train.LogProbs(x, torch.zeros(rows, dtype=torch.int32, device=cuda))
    s1 = 512 + (width - 512) * math.exp(-16.75)
    H = math.log(s1) + (width - 512) * math.exp(-16.75) * 16.75 / s1
    tol = u * (4 * H + 4 + 9 + 3 + 5) + 2 * u * math.log(s1)
    lost = math.log(s1 / 512)
    assert lost > 1.5 * tol
    assert float((r.LogSum.double() - math.log(s1)).abs().max()) <= tol
    assert float((r.LogProb.double() + math.log(s1)).abs().max()) <= tol


def test_clip_of_tensors_that_require_gradients(cuda):
    """Clipped alike whether their rows lie apart or not."""
    import torch

    from ai_b200 import train

    whole = _randn((20, 30), _gen(cuda, 3), cuda)
    apart = torch.zeros(20, 33, device=cuda)[:, :30].requires_grad_()
    apart.data.copy_(whole)
    whole.requires_grad_()
    assert float(train.ClipGradNorm([whole], 0.5)) == float(train.ClipGradNorm([apart], 0.5))
    assert torch.equal(whole, apart)
