"""The operators on the two ends of the vocabulary, ``token_logprobs`` and ``token_embedding``: values and gradients against
the formulas in float64, the conventions at the edges, layouts, and their refusals.

Tolerances.  u = 2^-24 is half a step of float32.  A sum of positive float32 terms is off by at most (additions on the way of
a term) * u relative.  A thread of the kernels adds at most 20 chunks of its own and one element besides, 81 terms of float32 and
161 of the two-byte types; a wave's sum is 6 additions more, the waves' at most 8, the parts' of a row that is cut 6 and a
factor: 178 u at most (98 u for float32).  An exponential is off by (3 + 2 |d|) u for its argument d (the instruction, the
rounding of the argument and of log2 e), weighted by its share in the sum; the mean of |d| so weighted is H less log Z, at
most 11 at 1310720 entries.  Together 203 u of Z (123 u for float32), of which the bounds' 220 u leave 17 for the logarithm and the
subtractions, beside their 4 u of |d| and of |log Z|.  The entropy's own sum of exp(d) d is off by the same additions of its
|log Z - H| and by 2 u of the mean of d squared, at most 130 u: less than 220 u (1 + |log Z - H|).  Results in a narrower type
are rounded once more, by half a step of that type."""
import ctypes

import numpy as np
import pytest
import torch

from pcfg_nat_amd import _lib, custom_ops as ops, harness, synth

U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]
# half the distance of neighbouring values next to zero (gfx950 keeps subnormal results of all three types; float32
# arithmetic on the way may flush below 2^-126)
SMALL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}
gpu = pytest.mark.gpu
DEV = "cuda"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------------
# the formulas in float64, row by row
# ------------------------------------------------------------------------------------------------------------------
def reference_row(x, top):
    """x: float64 [V] (numpy).  Returns (d = x - m, log Z, H, lp, ids)."""
    V = len(x)
    rank = np.where(np.isnan(x), np.inf, x)
    order = sorted(range(V), key=lambda i: (not np.isnan(x[i]), -rank[i] if not np.isnan(x[i]) else 0.0, i))[:top]
    if np.isnan(x).any() or np.isposinf(x).any():
        nan = np.full(V, np.nan)
        return nan, np.nan, np.nan, nan, order
    m = x.max()
    if np.isneginf(m):
        return np.full(V, -np.inf), -np.inf, 0.0, np.full(V, -np.inf), order
    d = x - m
    e = np.exp(d)
    Z = e.sum()
    lp = d - np.log(Z)
    H = np.log(Z) - (e[e > 0] * d[e > 0]).sum() / Z
    return d, np.log(Z), H, lp, order


def reference_grad(lp, H, ids, g):
    """ids, g: the entries that a gradient arrives at; g[0] of the entropy apart.  Returns (gradient, its float32 error bound)."""
    g_ent, entries = g
    p = np.exp(lp)
    G = sum(v for _, v in entries)
    A = sum(abs(v) for _, v in entries)
    live = np.where(p > 0, lp, 0.0)
    t = G + g_ent * (live + H)
    grad = -p * t
    arrived = np.zeros_like(p)
    for i, v in entries:
        grad[i] += v
        arrived[i] += abs(v)
    # p is off by the exponent's error relative, the bracket by the rounding of its parts, the entries by their additions
    off_lp = U * (4 * np.abs(live) + 220)
    bound = p * np.abs(t) * 2 * off_lp + p * (70 * U * A + abs(g_ent) * (off_lp + U * (220 * (2 + abs(H)) + 4 * np.abs(live)))) \
        + 70 * U * (arrived + p * np.abs(t)) + 2.0 ** -120 * (A + abs(g_ent) + 1)
    return grad, bound


def content(kind, rows, V, gen):
    x = torch.randn((rows, V), generator=gen) * 3.0
    if kind == "ties":
        x = torch.randint(-3, 4, (rows, V), generator=gen).float()
    elif kind == "constant":
        x = torch.full((rows, V), 1.5)
    elif kind == "zeros":
        x = torch.where(torch.rand((rows, V), generator=gen) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    elif kind == "masked":  # a few allowed entries, fewer than the alternatives asked for in some rows
        keep = torch.rand((rows, V), generator=gen) < min(0.5, 3.0 / V)
        x = x.masked_fill(~keep, float("-inf"))
    elif kind == "rising":
        x = torch.linspace(-8, 8, V).expand(rows, V).clone()
    elif kind == "falling":
        x = torch.linspace(8, -8, V).expand(rows, V).clone()
    elif kind == "block":  # all large entries next to each other
        x[:, V // 3:V // 3 + max(1, V // 8)] += 10.0
    elif kind == "large":
        x = x * 200.0
    return x


def check_logprobs(logits, tokens, top, got, grads=None):
    """Holds the results of one call on [rows, V] logits against the formulas.  grads: (grad_logits, g_lp, g_h, g_top)."""
    rows, V = logits.shape
    x = logits.detach().double().cpu().numpy()
    tok = None if tokens is None else tokens.cpu().tolist()
    out = [None if t is None else t.detach().double().cpu().numpy() for t in got]
    if grads is not None:
        dx, ups = grads[0].double().cpu().numpy(), [None if g is None else g.double().cpu().numpy() for g in grads[1:]]
        small, step = SMALL[logits.dtype], half_step(logits.dtype)
    for r in range(rows):
        if tok is not None and tok[r] < 0:
            assert out[0][r] == 0
            if out[1] is not None:
                assert out[1][r] == 0
            if top:
                assert (out[2][r] == -np.inf).all() and (out[3][r] == -1).all()
            if grads is not None:
                assert (dx[r] == 0).all()
            continue
        d, lz, H, lp, order = reference_row(x[r], top)
        empty = np.isneginf(lz)

        def near(value, i):
            # a log-probability below float32's lowest value, 2^128 (1 - 2^-24) = 3.4e38 away from zero, rounds to -inf: between the
            # largest and the lowest bfloat16 or float32 it is -6.8e38
            if lp[i] < -2.0 ** 128:
                return value == -np.inf
            if np.isnan(lp[i]):
                return np.isnan(value)
            return abs(value - lp[i]) <= U * (4 * abs(d[i]) + 4 * abs(lz) + 220)

        if tok is not None:
            if tok[r] >= V:
                assert np.isnan(out[0][r])
            else:
                assert near(out[0][r], tok[r]), (r, out[0][r], lp[tok[r]])
        if out[1] is not None:
            if np.isnan(H):
                assert np.isnan(out[1][r])
            else:
                bound = 0.0 if empty else U * (220 * (1 + abs(lz - H)) + 4 * abs(lz) + 4 * abs(H))
                assert abs(out[1][r] - H) <= bound, (r, out[1][r], H)
        if top:
            assert out[3][r].astype(int).tolist() == order, (r, out[3][r].astype(int).tolist(), order)
            for k in range(top):
                assert near(out[2][r][k], order[k]), (r, k)
        if grads is not None:
            entries = []
            if ups[0] is not None:
                entries.append((tok[r], ups[0][r]))
            if ups[2] is not None:
                entries += list(zip(order, ups[2][r]))
            if np.isnan(lz) or (ups[0] is not None and tok[r] >= V):
                assert np.isnan(dx[r]).all()
            elif empty:
                assert (dx[r] == 0).all()
            else:
                want, bound = reference_grad(lp, H, None, (0.0 if ups[1] is None else ups[1][r], entries))
                bound = bound + step * (np.abs(want) + bound) + small
                bad = np.abs(dx[r] - want) > bound
                assert not bad.any(), (r, int(bad.argmax()), dx[r][bad][:3], want[bad][:3], bound[bad][:3])


def run_logprobs(logits, tokens, top, entropy, train, gen):
    """One call on [rows, V] logits on the GPU (as they lie), checked; with its gradient where asked for."""
    if not train:
        got = ops.token_logprobs(logits, tokens, top=top, entropy=entropy)
        check_logprobs(logits, tokens, top, got)
        return got
    leaf = logits.detach().requires_grad_(True)
    got = ops.token_logprobs(leaf, tokens, top=top, entropy=entropy)
    ends = [got.logprobs, got.entropy, got.top_logprobs]
    ups = [None if e is None else torch.randn(e.shape, generator=gen).to(DEV) for e in ends]
    grad, = torch.autograd.grad([e for e in ends if e is not None], leaf, [u for u in ups if u is not None])
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    check_logprobs(logits, tokens, top, got, (grad, ups[0], ups[1], ups[2]))
    return got


def some_tokens(rows, V, gen, out_of_range=True):
    t = torch.randint(0, V, (rows,), generator=gen)
    if out_of_range and rows > 2:
        t[1] = -1
        t[2] = V
    return t.to(DEV)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 64, 65, 255, 513, 1000, 2049, 4100, 8200])
def test_logprobs_sizes(V, dtype):
    gen = torch.Generator().manual_seed(V)
    for rows, top in ((1, 0), (5, min(V, 1)), (4, min(V, 5)), (4, min(V, 64))):
        x = content("normal", rows, V, gen).to(dtype).to(DEV)
        print("logprobs V=%d rows=%d top=%d %s" % (V, rows, top, dtype), flush=True)
        run_logprobs(x, some_tokens(rows, V, gen), top, True, True, gen)
        run_logprobs(x, some_tokens(rows, V, gen), top, False, False, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["ties", "constant", "zeros", "masked", "rising", "falling", "block", "large"])
def test_logprobs_contents(kind, dtype):
    gen = torch.Generator().manual_seed(7)
    for V in (9, 300, 5000, 20011):
        for rows, top in ((6, min(V, 7)), (3, min(V, 64))):
            x = content(kind, rows, V, gen).to(dtype).to(DEV)
            print("logprobs %s V=%d top=%d %s" % (kind, V, top, dtype), flush=True)
            run_logprobs(x, some_tokens(rows, V, gen), top, True, True, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,V", [(1, 40000), (2, 33333), (3, 131072), (300, 40000), (2, 262147), (1100, 7001), (200, 90001)])
def test_logprobs_long_rows(rows, V, dtype):
    gen = torch.Generator().manual_seed(rows + V)
    x = (torch.randn((rows, V), generator=gen) * 3.0).to(dtype).to(DEV)
    tokens = some_tokens(rows, V, gen, out_of_range=False)
    print("logprobs rows=%d V=%d %s" % (rows, V, dtype), flush=True)
    got = ops.token_logprobs(x, tokens, top=20, entropy=True)
    some = slice(0, 3)
    check_logprobs(x[some], tokens[some], 20, [t[some] for t in got])
    if rows > 3:
        last = slice(rows - 2, rows)
        check_logprobs(x[last], tokens[last], 20, [t[last] for t in got])
    run_logprobs(x[some], tokens[some], 3, True, True, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [2500, 20003, 40000, 131075])
def test_logprobs_rows_whose_threshold_is_low(V, dtype):
    """Rows whose waves see very different elements, so that most of the row lies above the threshold that all of them agree
    on; with masks, a NaN or few entries left besides."""
    gen = torch.Generator().manual_seed(V)
    x = (torch.randn((6, V), generator=gen) * 3.0).to(dtype)
    width = 16 // x.element_size()
    low = ((torch.arange(V) // width) % 256 < 64).expand(6, V).clone()  # a wave's elements of four
    x = torch.where(low, x - 20, x)
    x[1] = x[1].masked_fill(low[1], float("-inf"))
    x[2] = x[2].masked_fill(low[2], torch.finfo(dtype).min)
    x[3, V // 2] = float("nan")
    few = torch.rand(V, generator=gen) < 8.0 / V
    x[4] = x[4].masked_fill(~few, float("-inf"))
    x[5] = x[5].masked_fill(~few, torch.finfo(dtype).min)
    x[4:, V // 3] = 1.0
    x = x.to(DEV)
    tokens = torch.full((6,), V // 3).to(DEV)
    for top in (1, 20, 64):
        print("logprobs, low threshold, V=%d top=%d %s" % (V, top, dtype), flush=True)
        run_logprobs(x, tokens, top, True, top == 20, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [5, 1500, 30001])
def test_logprobs_masked_infinite_and_nan(V, dtype):
    """Rows of nothing but -inf, of nothing but the type's lowest value, with the lowest value as the mask, with +inf, with
    a NaN, of nothing but NaN, with a single entry left."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((9, V), generator=gen).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = float("-inf")
    x[1] = low
    x[2, 1:] = low
    x[3, 2] = float("inf")
    x[4, V - 1] = float("nan")
    x[5] = float("nan")
    x[6] = float("-inf")
    x[6, V // 2] = 2.0
    x[7, ::2] = float("-inf")
    x[8, 1] = torch.finfo(dtype).max
    x[8, 2] = low
    tokens = torch.tensor([0, 1, 2, 2, 0, 1, V // 2, 0, 2]).to(DEV)
    for top in (0, 3, 5):
        run_logprobs(x.to(DEV), tokens, top, True, True, gen)
        run_logprobs(x.to(DEV), None, max(top, 1), True, False, gen)


def run_and_want_finite(logits, tokens, top, gen, arrives=None):
    """As run_logprobs with its gradient, of rows without NaN and +inf: nothing of the results is NaN but where a token lies beyond
    the vocabulary (a comparison with NaN holds nothing).  arrives: the gradient of every row's entropy, drawn otherwise."""
    leaf = logits.detach().requires_grad_(True)
    got = ops.token_logprobs(leaf, tokens, top=top, entropy=True)
    ups = [torch.randn(t.shape, generator=gen).to(DEV) for t in got[:3]]
    if arrives is not None:
        ups[1] = torch.full_like(ups[1], arrives)
    grad, = torch.autograd.grad(got[:3], leaf, ups)
    known = tokens < logits.size(1)
    assert not got.logprobs[known].isnan().any() and not got.entropy.isnan().any() and not got.top_logprobs.isnan().any()
    assert grad[known].isfinite().all()
    check_logprobs(logits, tokens, top, got, (grad, *ups))


FAR = [s * m for m in (1.6e7, 1e8, 1e10, 1e20, 1e29) for s in (1, -1)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("far", FAR, ids="{:.1e}".format)
def test_logprobs_far_from_zero(far, dtype):
    """Rows whose largest entry, or whose mask, lies far from zero, where the product of the maximum and log2 e is rounded by more
    than an exponent can hold: constant, one such entry among ordinary ones, a few ordinary ones among such, neighbouring values,
    half of the row one behind the other (whole parts of a row that is cut), -inf besides.  In one part and in three."""
    gen = torch.Generator().manual_seed(21)
    for V in (9, 300, 20011, 90001 if dtype == torch.bfloat16 else 45007):
        x = torch.randn((6, V), generator=gen) * 3.0
        few = torch.rand((V,), generator=gen) < 5.0 / V
        few[V // 2] = True
        x[0] = far
        x[1, V // 3] = far
        x[2] = x[2].masked_fill(~few, far)
        x[3] = far * (1.0 + torch.finfo(dtype).eps * torch.randint(0, 4, (V,), generator=gen))
        x[4, :V // 2] = far
        x[5] = far
        x[5, ::2] = float("-inf")
        x = x.to(dtype).to(DEV)
        top = min(V, 7)
        for tokens in (torch.full((6,), V // 3), torch.full((6,), V // 2), torch.tensor([0, 0, -1, V - 1, V - 1, V])):
            print("logprobs far=%g V=%d %s" % (far, V, dtype), flush=True)
            run_and_want_finite(x, tokens.to(DEV), top, gen)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("arrives", [1e6, 1e9, -1e12], ids="{:.0e}".format)
def test_logprobs_large_entropy_gradient(arrives, dtype):
    """A gradient of the entropy as large as a scaled loss makes it: entries without probability (-inf, the lowest value, a large
    negative number) have no gradient of their own, whatever arrives."""
    gen = torch.Generator().manual_seed(22)
    for V in (9, 300, 5000):
        masks = [float("-inf"), torch.finfo(dtype).min, -1e30, -1e10, -300.0]
        x = (torch.randn((len(masks), V), generator=gen) * 3.0).to(dtype)
        for r, mask in enumerate(masks):
            x[r, ::3] = mask
        run_and_want_finite(x.to(DEV), torch.full((len(masks),), V // 2).to(DEV), 3, gen, arrives)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_finite_inputs_give_finite_results(dtype):
    """No NaN out of numbers, masks and ordinary upstream gradients, over the ways in which both operators are launched."""
    gen = torch.Generator().manual_seed(23)
    for V in (1, 9, 300, 1001, 5000, 20011, 50021, 131075):
        for kind in ("normal", "constant", "masked", "block", "large"):
            x = content(kind, 5, V, gen).to(dtype)
            if V > 2:
                x[:, V - 1] = 0.5  # (an entry left in every row)
            print("logprobs %s V=%d %s" % (kind, V, dtype), flush=True)
            leaf = x.to(DEV).requires_grad_(True)
            got = ops.token_logprobs(leaf, torch.full((5,), V - 1).to(DEV), top=min(V, 6), entropy=True)
            ups = [torch.randn(t.shape, generator=gen).to(DEV) for t in got[:3]]
            grad, = torch.autograd.grad(got[:3], leaf, ups)
            # (a row of nothing but -inf, which a single masked entry is, has log-probabilities -inf)
            assert not got.logprobs.isnan().any() and not got.top_logprobs.isnan().any()
            assert got.entropy.isfinite().all() and grad.isfinite().all()
    for V, N, D in ((1, 1, 1), (300, 100, 5), (300, 8192, 16), (5000, 3001, 333), (40000, 5120, 512), (70001, 20000, 40), (3, 33000, 8)):
        weight = torch.randn((V, D), generator=gen).to(dtype).to(DEV).requires_grad_(True)
        tokens = torch.where(torch.rand((N,), generator=gen) < 0.4, torch.tensor(0), torch.randint(-1, V, (N,), generator=gen)).to(DEV)
        out = ops.token_embedding(weight, tokens, 2.0)
        grad, = torch.autograd.grad(out, weight, torch.full_like(out, 0.125))  # (no sum leaves float16)
        assert out.isfinite().all() and grad.isfinite().all(), (V, N, D)


def selections():
    """Rows whose alternatives were selected by reading the row again, since the last call of this."""
    torch.cuda.synchronize()
    rows = ctypes.c_ulonglong()
    _lib.check(_lib.load().pcfgnat_token_logprobs_selections(ctypes.byref(rows), 1), _lib.load())
    return rows.value


@gpu
@pytest.mark.parametrize("dtype,V", [(torch.float16, 1000), (torch.float16, 8000), (torch.bfloat16, 40000), (torch.float32, 40000),
                                     (torch.float16, 81921), (torch.bfloat16, 100277), (torch.float16, 122880), (torch.bfloat16, 131072),
                                     (torch.float32, 40961), (torch.float32, 50257), (torch.float32, 61441), (torch.float32, 250007),
                                     (torch.float32, 1310720)], ids=str)
def test_logprobs_ordinary_rows_take_the_threshold(dtype, V):
    """Alternatives of ordinary rows, in one part, in three and in more, of few rows and of many, come from the elements above the
    threshold of the waves' maxima, also where a mask of -inf or of the lowest value covers all but one part of the row; those
    of a constant row do not."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    selections()
    for rows in (1, 16, 191, 192):
        x = (torch.randn((rows, V), generator=gen, device=DEV) * 3.0).to(dtype)
        for top in (1, 20, 64):
            print("logprobs V=%d rows=%d top=%d %s" % (V, rows, top, dtype), flush=True)
            got = ops.token_logprobs(x, None, top=top, entropy=True)
            assert selections() == 0, (rows, top)
            if rows == 16 and top == 20:
                check_logprobs(x[:2], None, top, [None] + [t[:2] for t in got[1:]])
            if V < 40961:
                continue
            for low in (float("-inf"), torch.finfo(dtype).min):
                for cut in (slice(0, V // 3 + 64), slice(V // 4, V)):
                    y = x.clone()
                    y[:, cut] = low
                    got = ops.token_logprobs(y, None, top=top, entropy=True)
                    assert selections() == 0, (rows, top, low, cut)
                    if rows == 1 and top == 20:
                        check_logprobs(y, None, top, got)
        ops.token_logprobs(torch.full_like(x, 1.5), None, top=1)
        assert selections() == rows  # (more equal elements than a workgroup puts in order: 256 for one wave, 1024 for more)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_layouts(dtype):
    """Any alignment of a row, padded vocabularies, a batch without its first node, a transposed batch, an expanded row,
    one row as a vector, a strided vocabulary; shapes of the results; no rows at all."""
    gen = torch.Generator().manual_seed(11)
    V = 1003
    wide = torch.randn((6, V + 17), generator=gen).to(dtype).to(DEV)
    for off in range(9):
        run_logprobs(wide[:, off:off + V], some_tokens(6, V, gen), 4, True, True, gen)
    cube = torch.randn((4, 5, V + 3), generator=gen).to(dtype).to(DEV)
    row = torch.randn((1, V), generator=gen).to(dtype).to(DEV)
    for x in (cube[:, 1:, :V], cube.transpose(0, 1)[:, :, :V], cube[::2, ::3, 2:V + 2], row.expand(7, V), cube[1, 2, :V],
              cube.transpose(0, 2)[:V], cube.unsqueeze(1).expand(4, 3, 5, V + 3)[..., :V], cube[None, :, None, 2:4, :V]):
        lead = x.shape[:-1]
        tokens = torch.randint(0, x.size(-1), lead, generator=gen).to(DEV)
        leaf = x.detach().requires_grad_(True)
        top = min(3, x.size(-1))
        got = ops.token_logprobs(leaf, tokens, top=top, entropy=True)
        assert got.logprobs.shape == lead and got.entropy.shape == lead
        assert got.top_logprobs.shape == lead + (top,) and got.top_tokens.shape == lead + (top,)
        ups = [torch.randn(t.shape, generator=gen).to(DEV) for t in got[:3]]
        grad, = torch.autograd.grad(got[:3], leaf, ups)
        assert grad.shape == x.shape
        flat = x.reshape(-1, x.size(-1))
        check_logprobs(flat, tokens.reshape(-1), top, [t.reshape(flat.size(0), *t.shape[len(lead):]) for t in got],
                       (grad.reshape(flat.shape), *[u.reshape(flat.size(0), *u.shape[len(lead):]) for u in ups]))
    tokens = some_tokens(6, V, gen)
    spaced = torch.stack([tokens, tokens], 1)[:, 0]
    assert spaced.stride(0) == 2
    run_logprobs(wide[:, :V], spaced, 0, True, True, gen)
    empty = torch.empty((3, 0, 7), dtype=dtype, device=DEV, requires_grad=True)
    ops.token_logprobs(empty, torch.empty((3, 0), dtype=torch.int64, device=DEV), top=2).logprobs.sum().backward()
    assert empty.grad.shape == (3, 0, 7)
    none = ops.token_logprobs(torch.empty((0, 4, 7), dtype=dtype, device=DEV), torch.empty((0, 4), dtype=torch.int64, device=DEV), top=2)
    assert none.logprobs.shape == (0, 4) and none.top_tokens.shape == (0, 4, 2) and none.entropy is None


@gpu
def test_logprobs_gradient_by_parts_and_by_differences():
    """Each of the three results alone gives its part of the gradient; the whole against central differences in float64 of
    the formula; a token that is also an alternative; an expanded and a strided upstream gradient."""
    gen = torch.Generator().manual_seed(5)
    V, rows, top = 37, 3, 5
    x = (torch.randn((rows, V), generator=gen) * 2).to(DEV)
    tokens = x.argmax(-1)  # every token is its row's first alternative

    def value(y, a, b, c):
        lp = torch.log_softmax(y, -1)
        ids = y.sort(dim=-1, descending=True, stable=True).indices[:, :top]
        return (a * lp.gather(-1, tokens.cpu()[:, None])[:, 0]).sum() + (b * -(lp.exp() * lp).sum(-1)).sum() + (c * lp.gather(-1, ids)).sum()

    parts = []
    a, b, c = (torch.randn(s, generator=gen) for s in ((rows,), (rows,), (rows, top)))
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        leaf = x.clone().requires_grad_(True)
        got = ops.token_logprobs(leaf, tokens, top=top, entropy=True)
        loss = sum((w.to(DEV) * t).sum() for w, t, on in zip((a, b, c), got[:3], which) if on)
        loss.backward()
        parts.append(leaf.grad.double().cpu())
        y = x.double().cpu()
        want = torch.zeros_like(y)
        h = 1e-5
        wa, wb, wc = (w.double() * on for w, on in zip((a, b, c), which))
        for r in range(rows):
            for v in range(V):
                up, down = y.clone(), y.clone()
                up[r, v] += h
                down[r, v] -= h
                want[r, v] = (value(up, wa, wb, wc) - value(down, wa, wb, wc)) / (2 * h)
        # float32 arithmetic on gradients of size 1..10: 2^-24 * 220 * 10; the differences themselves: h^2 and 1e-16 / h
        assert (parts[-1] - want).abs().max() <= 220 * U * 10 + 1e-7
    assert (parts[0] + parts[1] + parts[2] - parts[3]).abs().max() <= 220 * U * 10
    leaf = x.clone().requires_grad_(True)
    ops.token_logprobs(leaf, tokens).logprobs.sum().backward()  # an expanded upstream gradient
    p = torch.softmax(x.double(), -1)
    p.scatter_add_(1, tokens[:, None], -torch.ones((rows, 1), dtype=torch.float64, device=DEV))
    assert (leaf.grad.double() + p).abs().max() <= 220 * U
    got = ops.token_logprobs(leaf, tokens, top=top, entropy=True)  # twice through one graph: the same bits
    loss = got.logprobs.sum() + got.entropy.sum() + got.top_logprobs.sum()
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    second, = torch.autograd.grad(loss, leaf)
    assert torch.equal(first, second)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_agree_with_the_front_end(dtype):
    """The first alternative is what the decode's front-end (logsoftmax_max) finds."""
    if dtype == torch.bfloat16:
        pytest.skip("logsoftmax_max takes no bfloat16")
    gen = torch.Generator().manual_seed(9)
    x = (torch.randn((3, 20, 4000), generator=gen) * 3).to(dtype).to(DEV)
    best, idx = ops.logsoftmax_max(x)
    got = ops.token_logprobs(x, idx, top=1)
    assert torch.equal(got.top_tokens[..., 0], idx)
    assert (got.top_logprobs[..., 0] - best).abs().max() <= 2 * U * 240
    assert torch.equal(got.logprobs, got.top_logprobs[..., 0])


# ------------------------------------------------------------------------------------------------------------------
# token_embedding
# ------------------------------------------------------------------------------------------------------------------
def check_embedding(weight, tokens, scale, pad, out, up=None, grad=None):
    V, D = weight.shape
    w, t = weight.detach().double().cpu(), tokens.reshape(-1).cpu()
    s = float(np.float32(scale))
    step, small = half_step(weight.dtype), SMALL[weight.dtype]
    want = w[t.clamp(0, V - 1)] * s
    want[t < 0] = 0.0
    got = out.detach().double().cpu().reshape(-1, D)
    assert torch.isnan(got[t >= V]).all()
    live = t < V
    err = (got - want).abs() - ((step + 2 * U) * want.abs() + small)
    assert not (err[live] > 0).any()
    if grad is None:
        return
    g = up.double().cpu().reshape(-1, D)
    keep = (t >= 0) & (t < V) & (t != (-1 if pad is None else pad))
    want = torch.zeros((V, D), dtype=torch.float64).index_add_(0, t[keep], g[keep]) * s
    mass = torch.zeros((V, D), dtype=torch.float64).index_add_(0, t[keep], g[keep].abs()) * abs(s)
    count = torch.zeros((V,), dtype=torch.float64).index_add_(0, t[keep], torch.ones_like(t[keep], dtype=torch.float64))
    bound = (count[:, None] + 2) * U * mass
    bound = bound + step * (want.abs() + bound) + small
    got = grad.double().cpu()
    bad = (got - want).abs() > bound
    assert not bad.any(), (bad.nonzero()[:3], got[bad][:3], want[bad][:3], bound[bad][:3])
    assert (got[count == 0] == 0).all()


def run_embedding(V, D, tokens, dtype, scale, pad, gen, weight=None):
    weight = (torch.randn((V, D), generator=gen).to(dtype).to(DEV) if weight is None else weight)
    plain = ops.token_embedding(weight, tokens, scale=scale, padding_idx=pad)
    assert plain.dtype == dtype and plain.shape == tokens.shape + (D,)
    leaf = weight.detach().requires_grad_(True)
    out = ops.token_embedding(leaf, tokens, scale=scale, padding_idx=pad)
    assert torch.equal(out.detach().nan_to_num(7.0), plain.nan_to_num(7.0))
    up = torch.randn(out.shape, generator=gen).to(dtype).to(DEV)
    grad, = torch.autograd.grad(out, leaf, up)
    assert grad.dtype == dtype and grad.shape == weight.shape
    check_embedding(weight, tokens, scale, pad, out, up, grad)
    return grad


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 2, 3, 7, 8, 31, 64, 130, 512, 515, 1024, 2056])
def test_embedding_sizes(D, dtype):
    gen = torch.Generator().manual_seed(D)
    for V, N in ((1, 1), (5, 3), (67, 130), (300, 1000), (300, 8193)):
        tokens = torch.randint(-1, V + 1, (N,), generator=gen).to(DEV)
        print("embedding V=%d N=%d D=%d %s" % (V, N, D, dtype), flush=True)
        run_embedding(V, D, tokens, dtype, 1.0, None, gen)
        run_embedding(V, D, tokens, dtype, D ** 0.5, 0, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N,D", [(4099, 72), (5000, 523), (9000, 72), (17001, 8)])  # (in one, three, three and four launches)
@pytest.mark.parametrize("kind", ["one", "two", "runs", "every", "reversed", "none", "pads", "ends"])
def test_embedding_token_distributions(kind, N, D, dtype):
    """One token everywhere, two taking turns, runs, every row once, in reverse, no row at all, nearly all padding, the
    first and the last row."""
    gen = torch.Generator().manual_seed(2)
    V = N
    i = torch.arange(N)
    t = {"one": torch.full((N,), 17), "two": 5 + 4000 * (i % 2), "runs": i // 97, "every": i.clone(), "reversed": V - 1 - i,
         "none": torch.where(i % 2 == 0, torch.tensor(-1), torch.tensor(V)),
         "pads": torch.where(i % 50 == 0, i, torch.tensor(1)), "ends": (i % 2) * (V - 1)}[kind]
    run_embedding(V, D, t.to(DEV), dtype, 3.0, 1, gen)


@gpu
@pytest.mark.parametrize("V,N", [(40000, 5120), (257, 70000), (250007, 3), (3, 33000), (70001, 20000), (300000, 50), (2, 8192), (65537, 8192), (300000, 20000), (256, 16385), (262144, 18433)])
def test_embedding_large(V, N):
    gen = torch.Generator().manual_seed(V)
    t = torch.where(torch.rand((N,), generator=gen) < 0.4, torch.tensor(min(3, V - 1)), torch.randint(0, V, (N,), generator=gen))
    print("embedding V=%d N=%d" % (V, N), flush=True)
    run_embedding(V, 16, t.to(DEV), torch.float16, 4.0, 1, gen)
    run_embedding(V, 33, t.to(DEV), torch.float32, 1.0, None, gen)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embedding_layouts(dtype):
    """Batched and strided tokens, rows of a wider weight, a weight at an odd offset, a transposed weight, expanded and
    transposed upstream gradients, no tokens at all; the same inputs give the same bits."""
    gen = torch.Generator().manual_seed(4)
    V, D = 50, 24
    batch = torch.randint(0, V, (3, 7, 2), generator=gen).to(DEV)
    run_embedding(V, D, batch, dtype, 2.0, 1, gen)
    run_embedding(V, D, batch.transpose(0, 1), dtype, 2.0, 1, gen)
    run_embedding(V, D, torch.tensor(3, device=DEV), dtype, 2.0, 1, gen)
    wide = torch.randn((V, D + 9), generator=gen).to(dtype).to(DEV)
    for off in (0, 1, 3, 8):
        run_embedding(V, D, batch, dtype, 2.0, 1, gen, weight=wide[:, off:off + D])
    run_embedding(V, D, batch, dtype, 2.0, 1, gen, weight=torch.randn((D, V), generator=gen).to(dtype).to(DEV).t())
    flat = batch.reshape(-1)
    weight = torch.randn((V, D), generator=gen).to(dtype).to(DEV).requires_grad_(True)
    up = torch.randn((D, flat.numel()), generator=gen).to(dtype).to(DEV).t()
    base = torch.randn((flat.numel(), D + 5), generator=gen).to(dtype).to(DEV)
    for g in (up, up[:1].expand(flat.numel(), D), up[:, :1].expand(flat.numel(), D), base[:, 3:3 + D], base[:1, :D].expand(flat.numel(), D)):
        out = ops.token_embedding(weight, flat, 2.0, 1)
        grad, = torch.autograd.grad(out, weight, g)
        check_embedding(weight, flat, 2.0, 1, out, g, grad)
        again, = torch.autograd.grad(ops.token_embedding(weight, flat, 2.0, 1), weight, g)
        assert torch.equal(grad, again)
    ops.token_embedding(weight, flat, 2.0).sum().backward()
    none = torch.empty((0, 4), dtype=torch.int64, device=DEV)
    weight.grad = None
    out = ops.token_embedding(weight, none, 2.0)
    assert out.shape == (0, 4, D)
    out.sum().backward()
    assert (weight.grad == 0).all()


# ------------------------------------------------------------------------------------------------------------------
# both, as they would be used
# ------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_tied_weight_gradient_from_both_ends(dtype):
    """Embedding and vocabulary projection share one matrix: tokens in, log-probabilities, entropy and alternatives out, one
    backward; against autograd over the plain formulas in float64 on the same (rounded) intermediate values."""
    gen = torch.Generator().manual_seed(6)
    V, D, B, L = 301, 32, 3, 11
    weight = (torch.randn((V, D), generator=gen) * 0.3).to(dtype).to(DEV).requires_grad_(True)
    tokens = torch.randint(0, 40, (B, L), generator=gen).to(DEV)
    targets = torch.randint(0, V, (B, L), generator=gen).to(DEV)
    targets[:, -2:] = -1
    h = ops.token_embedding(weight, tokens, scale=2.0, padding_idx=1)
    logits = h @ weight.t()
    got = ops.token_logprobs(logits, targets, top=2, entropy=True)
    loss = -got.logprobs.sum() - 0.1 * got.entropy.sum() + 0.5 * got.top_logprobs.masked_fill(targets[..., None] < 0, 0.0).sum()
    loss.backward()
    w = weight.detach().double().cpu().requires_grad_(True)
    e = w[tokens.cpu()] * 2.0
    e = torch.where(tokens.cpu()[..., None] == 1, e.detach(), e)
    e = e + (h.detach().double().cpu() - e).detach()
    y = e @ w.t()
    y = y + (logits.detach().double().cpu() - y).detach()  # the values of the rounded path, the derivative of the exact one
    y.retain_grad()
    lp = torch.log_softmax(y, -1)
    live = (targets >= 0).cpu()
    ids = y.sort(dim=-1, descending=True, stable=True).indices[..., :2]
    assert torch.equal(got.top_tokens.cpu()[live], ids[live])
    tl = lp.gather(-1, targets.cpu().clamp(min=0)[..., None])[..., 0]
    ent = -(lp.exp() * lp).sum(-1)
    want = -tl[live].sum() - 0.1 * ent[live].sum() + 0.5 * lp.gather(-1, ids)[live].sum()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 240 * U * float(live.sum()) * 30
    # each part of the gradient is a sum of products of rounded factors: the logits' gradient and the embeddings' rounded once
    # each, then the part and the sum of the parts, four half steps of the summed magnitudes; 800 u for the arithmetic in
    # float32 (sums of up to 301 terms, probabilities as in reference_grad)
    dl, wa = y.grad.abs().reshape(-1, V), w.detach().abs()
    mass = dl.t() @ e.detach().abs().reshape(-1, D)
    mass.index_add_(0, tokens.cpu().reshape(-1), (dl @ wa) * 2.0)
    err = (weight.grad.double().cpu() - w.grad).abs()
    assert not (err > (4 * half_step(dtype) + 800 * U) * mass + 8 * SMALL[dtype]).any()


@gpu
@pytest.mark.parametrize("single_call", [False, True])
def test_glancing_step_with_its_embeddings(single_call):
    """The GLAT step with ``embed``: the tokens as without it, and the embeddings that the decoder takes next."""
    batch = synth.config1()
    B, L, V = batch["logits"].shape
    prev = torch.full((B, L), 3, dtype=torch.int64)
    prev[1, 24:] = synth.PAD
    weight = torch.randn((V, 16), generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_(True)
    args = (batch["targets"].to(DEV), prev.to(DEV), batch["links"].to(DEV), 0.5)
    outs = []
    for embed in (None, (weight, 4.0)):
        outs.append(harness.glat_alignment(batch["logits"].clone().to(DEV), *args, generator=torch.Generator().manual_seed(7),
                                           noise_device="cpu", single_call=single_call, embed=embed))
    for key, value in outs[0].items():
        assert torch.equal(outs[1][key], value)
    glanced = outs[1]["glat_prev_output_tokens"]
    up = torch.randn((B, L, 16), generator=torch.Generator().manual_seed(2)).to(DEV)
    grad, = torch.autograd.grad(outs[1]["decoder_input"], weight, up)
    check_embedding(weight, glanced, 4.0, synth.PAD, outs[1]["decoder_input"], up, grad)
    assert (grad[synth.PAD] == 0).all()


@gpu
@pytest.mark.parametrize("alternatives", [1, 6])
def test_decode_with_alternatives(alternatives):
    """The decode whose front-end also gives every node's alternatives: tokens and lengths as by the Viterbi decode over the
    first alternatives, the same tokens as the model's own front-end finds, the alternatives those of the formulas."""
    logits, links, ol, mask = (t.to(DEV) for t in _decode_case())
    tokens, length, nodes = harness.decode_from_logits(logits, links, ol, mask, alternatives=alternatives)
    best, idx = ops.logsoftmax_max(logits)
    assert torch.equal(nodes.top_tokens[..., 0], idx) and (nodes.top_logprobs[..., 0] - best).abs().max() <= 2 * U * 240
    want_tokens, want_length = harness.viterbi_decode(nodes.top_logprobs[..., 0].contiguous(), idx, links, ol, mask, single_call=True)
    assert torch.equal(tokens, want_tokens) and torch.equal(length, want_length)
    rows = logits.shape[0] * logits.shape[1]
    check_logprobs(logits.reshape(rows, -1), None, alternatives, [None, nodes.entropy.reshape(rows)] + [t.reshape(rows, alternatives) for t in nodes[2:]])


def _decode_case():
    batch = synth.decode_batch([8, 5, 7], seed=3, V=700)
    mask, _, _ = synth.support_masks(batch["logits"].shape[1], 1)
    return batch["logits"], batch["links"], batch["output_length"], mask


# ------------------------------------------------------------------------------------------------------------------
# streams, graphs, far offsets, the C-ABI
# ------------------------------------------------------------------------------------------------------------------
def _step(logits, tokens, weight, words, ups):
    """A forward and backward of both operators; all results."""
    got = ops.token_logprobs(logits, tokens, top=3, entropy=True)
    dx, = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], logits, ups[:3])
    out = ops.token_embedding(weight, words, scale=2.0, padding_idx=1)
    dw, = torch.autograd.grad(out, weight, ups[3])
    return [t.detach() for t in got] + [dx, out.detach(), dw]


def _step_inputs(seed, V, rows=37):
    N = 300 if V < 10000 else 20000  # (the gradient of the embedding in one launch, in four)
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((rows, V), generator=gen).half().to(DEV).requires_grad_(True)
    tokens = torch.randint(-1, V, (rows,), generator=gen).to(DEV)
    weight = torch.randn((500, 24), generator=gen).half().to(DEV).requires_grad_(True)
    words = torch.where(torch.rand((N,), generator=gen) < 0.5, torch.tensor(3), torch.randint(0, 500, (N,), generator=gen)).to(DEV)
    ups = [torch.randn(s, generator=gen).to(DEV) for s in ((rows,), (rows,), (rows, 3))] + [torch.randn((N, 24), generator=gen).half().to(DEV)]
    return logits, tokens, weight, words, ups


@gpu
@pytest.mark.parametrize("V", [1001, 90001])
def test_on_another_stream_and_from_threads(V):
    """The same results, bit for bit, on a stream of its own behind work that the inputs wait for, and from two threads on two
    streams at once."""
    import threading
    args = [_step_inputs(s, V) for s in (1, 2)]
    want = [_step(*a) for a in args]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    source = args[0][0].detach().clone()
    late = torch.zeros_like(source)
    with torch.cuda.stream(side):
        big = torch.ones((4096, 4096), device=DEV)
        for _ in range(4):
            big = big @ big * 1e-4
        late.copy_(source)
        got = _step(late.requires_grad_(True), *args[0][1:])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    results, errors = [[], []], []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    results[k].append(_step(*args[k]))
            stream.synchronize()
        except Exception as e:  # (shown by the assertion below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k in range(2):
        for r in results[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


@gpu
@pytest.mark.parametrize("V", [1001, 90001])
def test_captured_into_graphs(V):
    """Forward and backward of both operators captured, two graphs out of one memory pool: replayed in turn with new inputs in
    place and eager work between, every replay the eager results bit for bit."""
    sets = [_step_inputs(s, V) for s in (3, 4)]
    fresh = [_step_inputs(s, V) for s in (5, 6, 7)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in sets:
            _step(*a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(_step(*a))
        graphs.append(g)
    for turn, new in enumerate(fresh):
        for k in range(2):
            with torch.no_grad():
                for into, value in zip(sets[k][:4], new[:4]):
                    into.copy_(value)
                for into, value in zip(sets[k][4], new[4]):
                    into.copy_(value)
            graphs[k].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs[k]]
            want = _step(*new)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (turn, k)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 bytes and 2^31 elements of logits, of their gradient and of a weight: the last rows."""
    gen = torch.Generator().manual_seed(8)
    rows, V = 54000, 40000
    assert rows * V > 2 ** 31
    logits = torch.zeros((rows, V), dtype=torch.float16, device=DEV)
    tail = (torch.randn((3, V), generator=gen) * 2).half().to(DEV)
    logits[-3:] = tail
    tokens = torch.full((rows,), -1, dtype=torch.int64, device=DEV)
    tokens[-3:] = torch.tensor([0, V - 1, 77], device=DEV)
    leaf = logits.requires_grad_(True)
    got = ops.token_logprobs(leaf, tokens, top=4, entropy=True)
    ups = [torch.randn(t.shape, generator=gen).to(DEV) for t in got[:3]]
    grad, = torch.autograd.grad(got[:3], leaf, ups)
    assert (grad[:3] == 0).all() and (grad[rows // 2] == 0).all()
    check_logprobs(tail, tokens[-3:], 4, [t[-3:] for t in got], (grad[-3:], *[u[-3:] for u in ups]))
    del leaf, logits, grad, got
    torch.cuda.empty_cache()
    V, D = 1100000, 2048
    assert V * D > 2 ** 31
    weight = torch.zeros((V, D), dtype=torch.float16, device=DEV)
    weight[-2:] = torch.randn((2, D), generator=gen).half().to(DEV)
    words = torch.tensor([V - 1, 0, V - 2, V - 1], device=DEV)
    leaf = weight.requires_grad_(True)
    out = ops.token_embedding(leaf, words, scale=3.0)
    up = torch.randn((4, D), generator=gen).half().to(DEV)
    grad, = torch.autograd.grad(out, leaf, up)
    short = torch.cat([weight.detach()[:1], weight.detach()[-2:]])
    check_embedding(short, torch.tensor([2, 0, 1, 2]), 3.0, None, out, up, torch.cat([grad[:1], grad[-2:]]))
    assert not grad[1:-2].any()
    del leaf, weight, grad, out
    torch.cuda.empty_cache()


@gpu
def test_more_rows_than_a_grid_dimension_has_waves():
    """70 million rows of two entries: a wave each is more than 2^32 threads.  Whole results against the formulas."""
    rows = 70000001
    x = torch.randn((rows, 2), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    tokens = torch.ones((rows,), dtype=torch.int64, device=DEV)
    tokens[12345::1000] = -1
    leaf = x.requires_grad_(True)
    lp = ops.token_logprobs(leaf, tokens).logprobs
    grad, = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
    live = tokens >= 0
    d = (x.detach()[:, 0].float() - x.detach()[:, 1].float())
    want = torch.where(live, -torch.nn.functional.softplus(d), torch.zeros_like(d))
    # |log-probability| < 20 here: its own rounding and that of the comparison's formula, U (4 d + 220) each
    assert (lp.detach() - want).abs().max() <= 2 * U * 300
    p = torch.where(live, torch.sigmoid(d), torch.zeros_like(d))
    for column, sign in ((0, -1.0), (1, 1.0)):
        assert (grad[:, column].float() - sign * p).abs().max() <= half_step(torch.float16) + 2 * U * 600
    del x, leaf, tokens, lp, grad, want, p, d, live
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("N", [64, 8200])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_c_abi_with_results_at_any_element(dtype, N):
    """The entry points called directly, their results one element behind an aligned address; what lies around them stays."""
    lib = _lib.load()
    gen = torch.Generator().manual_seed(12)
    code = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    rows, V = 5, 3001
    x = torch.randn((rows, V), generator=gen).to(dtype).to(DEV)
    tokens = some_tokens(rows, V, gen)
    f = lambda *shape: torch.full(shape, 7.0, device=DEV)  # noqa: E731
    lp, h, tl, stats = f(rows), f(rows), f(rows, 2), f(3, rows)
    tt = torch.zeros((rows, 2), dtype=torch.int64, device=DEV)
    _lib.check(lib.pcfgnat_token_logprobs(x.data_ptr(), code, 1, rows, 0, V, tokens.data_ptr(), lp.data_ptr(), h.data_ptr(), 2, tl.data_ptr(),
                                          tt.data_ptr(), stats.data_ptr(), None, V, stream), lib)
    guard = torch.full((rows * V + 2,), 7.0, dtype=dtype, device=DEV)
    ups = [torch.randn(s, generator=gen).to(DEV) for s in ((rows,), (rows,), (rows, 2))]
    _lib.check(lib.pcfgnat_token_logprobs_backward(x.data_ptr(), code, 1, rows, 0, V, tokens.data_ptr(), tt.data_ptr(), 2, stats.data_ptr(),
                                                   ups[0].data_ptr(), ups[1].data_ptr(), ups[2].data_ptr(), guard[1:].data_ptr(), V, stream), lib)
    assert guard[0] == 7 and guard[-1] == 7
    check_logprobs(x, tokens, 2, (lp, h, tl, tt), (guard[1:-1].view(rows, V), *ups))
    vocab, D = 40, 29
    weight = torch.randn((vocab, D), generator=gen).to(dtype).to(DEV)
    words = torch.randint(0, vocab // 2, (N,), generator=gen).to(DEV)
    out = torch.full((N * D + 2,), 7.0, dtype=dtype, device=DEV)
    _lib.check(lib.pcfgnat_token_embedding(weight.data_ptr(), code, D, words.data_ptr(), 2.0, out[1:].data_ptr(), N, vocab, D, stream), lib)
    dw = torch.full((vocab * D + 2,), 7.0, dtype=dtype, device=DEV)
    up = torch.randn((N, D), generator=gen).to(dtype).to(DEV)
    need = lib.pcfgnat_token_embedding_backward_workspace_bytes(code, N, vocab, D)
    assert (need == 0) == (N <= 8192)
    work = torch.full((need + 16,), 85, dtype=torch.uint8, device=DEV)
    _lib.check(lib.pcfgnat_token_embedding_backward(up.data_ptr(), code, D, words.data_ptr(), 2.0, -1, dw[1:].data_ptr(), work.data_ptr(), N, vocab,
                                                    D, stream), lib)
    for t in (out, dw):
        assert t[0] == 7 and t[-1] == 7
    assert (work[need:] == 85).all()
    check_embedding(weight, words, 2.0, None, out[1:-1].view(N, D), up, dw[1:-1].view(vocab, D))


# ------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------
def test_refusals_without_a_gpu():
    z = torch.zeros
    t = z((2,), dtype=torch.int64)
    for call, what in ((lambda: ops.token_logprobs(z(2, 5), t), "GPU"),
                       (lambda: ops.token_logprobs(z(2, 5)), "nothing is asked for"),
                       (lambda: ops.token_logprobs(z(2, 5, dtype=torch.float64), t), "dtype"),
                       (lambda: ops.token_logprobs(z(2, 5, dtype=torch.int64), t), "dtype"),
                       (lambda: ops.token_logprobs(z(2, 5), t.int()), "long"),
                       (lambda: ops.token_logprobs(z(2, 5), z((3,), dtype=torch.int64)), "shape"),
                       (lambda: ops.token_logprobs(z(2, 5), z((2, 1), dtype=torch.int64)), "shape"),
                       (lambda: ops.token_logprobs(z(2, 5), t, top=6), "top must be"),
                       (lambda: ops.token_logprobs(z(2, 500), t, top=65), "top must be"),
                       (lambda: ops.token_logprobs(z(2, 5), t, top=-1), "top must be"),
                       (lambda: ops.token_logprobs(z(2, 0), t, entropy=True), "vocab"),
                       (lambda: ops.token_logprobs(torch.tensor(1.0), entropy=True), "vocab"),
                       (lambda: ops.token_embedding(z(4, 3), t), "GPU"),
                       (lambda: ops.token_embedding(z(4, 3, dtype=torch.float64), t), "dtype"),
                       (lambda: ops.token_embedding(z(4), t), "weight must be"),
                       (lambda: ops.token_embedding(z(0, 3), t), "weight must be"),
                       (lambda: ops.token_embedding(z(4, 0), t), "weight must be"),
                       (lambda: ops.token_embedding(z(4, 3), t.int()), "long"),
                       (lambda: ops.token_embedding(z(4, 3), t, padding_idx=4), "padding_idx"),
                       (lambda: ops.token_embedding(z(4, 3), t, padding_idx=-1), "padding_idx")):
        with pytest.raises(RuntimeError, match=what):
            call()


def test_c_abi_refusals_without_a_gpu():
    lib = _lib.load()
    one = 16  # an address that is never read: sizes are checked first

    def refused(rc, what):
        assert rc == _lib.EINVAL and what in lib.pcfgnat_last_error(), lib.pcfgnat_last_error()

    def logprobs(dtype=_lib.F16, outer=1, inner=2, V=8, top=0, logits=one, tokens=one, lp=one, tl=one, tt=one):
        return lib.pcfgnat_token_logprobs(logits, dtype, outer, inner, 16, 8, tokens, lp, None, top, tl, tt, None, None, V, None)

    refused(logprobs(dtype=_lib.F64), b"float16, bfloat16 or float32")
    refused(logprobs(V=0), b"dimensions")
    refused(logprobs(outer=-1), b"dimensions")
    refused(logprobs(outer=1 << 20, inner=1 << 20), b"dimensions")
    refused(logprobs(V=64 * 256 * 20 * 4 + 1), b"vocabulary of at most")
    refused(logprobs(top=9), b"alternatives")
    refused(logprobs(top=65, V=100), b"alternatives")
    refused(logprobs(logits=None), b"null")
    refused(logprobs(lp=None), b"null")
    refused(logprobs(tokens=None), b"null")
    refused(logprobs(top=1, tt=None), b"null")
    assert logprobs(outer=0) == _lib.OK  # no rows are no work

    def grad(dtype=_lib.F16, V=8, top=0, stats=one, tokens=one, tt=None, g=one, gt=None, out=one):
        return lib.pcfgnat_token_logprobs_backward(one, dtype, 1, 2, 16, 8, tokens, tt, top, stats, g, None, gt, out, V, None)

    refused(grad(dtype=9), b"float16, bfloat16 or float32")
    refused(grad(V=-3), b"dimensions")
    refused(grad(stats=None), b"null")
    refused(grad(tokens=None), b"null")
    refused(grad(out=None), b"null")
    refused(grad(top=2, gt=one), b"null")

    def embed(dtype=_lib.F16, stride=4, N=2, V=8, D=4, weight=one, tokens=one, out=one):
        return lib.pcfgnat_token_embedding(weight, dtype, stride, tokens, 1.0, out, N, V, D, None)

    refused(embed(dtype=_lib.F64), b"float16, bfloat16 or float32")
    refused(embed(stride=3), b"dimensions")
    refused(embed(V=0), b"dimensions")
    refused(embed(D=0), b"dimensions")
    refused(embed(N=-1), b"dimensions")
    refused(embed(N=1 << 25, D=1 << 14, stride=1 << 14), b"too large")
    refused(embed(weight=None), b"null")
    assert embed(N=0) == _lib.OK

    def embed_grad(dtype=_lib.F16, N=2, V=8, D=4, g=one, tokens=one, out=one, ws=one):
        return lib.pcfgnat_token_embedding_backward(g, dtype, D, tokens, 1.0, -1, out, ws, N, V, D, None)

    refused(embed_grad(dtype=_lib.F64), b"float16, bfloat16 or float32")
    refused(embed_grad(V=0), b"dimensions")
    refused(embed_grad(N=(16 << 22) + 1), b"dimensions")
    refused(embed_grad(N=1 << 26, D=1 << 20), b"too large")
    refused(embed_grad(g=None), b"null")
    refused(embed_grad(out=None), b"null")
    refused(embed_grad(N=9000, ws=None), b"null")
    refused(embed_grad(N=8000, D=600, ws=None), b"null")
    assert lib.pcfgnat_token_embedding_backward_workspace_bytes(_lib.F16, 51, 40000, 512) == 0  # in one launch
    assert lib.pcfgnat_token_embedding_backward_workspace_bytes(_lib.F16, 51200, 40000, 512) > 0


@gpu
def test_refusals_on_the_gpu():
    x = torch.zeros((2, 5), device=DEV, requires_grad=True)
    t = torch.zeros((2,), dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.token_logprobs(x, t.cpu())
    lp = ops.token_logprobs(x, t).logprobs
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(lp.sum(), x, create_graph=True)
    w = torch.zeros((4, 3), device=DEV, requires_grad=True)
    out = ops.token_embedding(w, t)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out.sum(), w, create_graph=True)
    y = x * 1.0
    lp = ops.token_logprobs(y, t).logprobs
    y.add_(1.0)  # the logits are read again by the backward
    with pytest.raises(RuntimeError, match="inplace"):
        lp.sum().backward()
