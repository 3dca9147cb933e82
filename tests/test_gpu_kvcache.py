"""Key/value cache operators (nwc_b200.KVCache) against the 64-bit restatement of tests/kv_reference.py.

Error bounds (half steps: bf16 2^-8, e4m3 2^-4, fp32 2^-24 relative).
Stored rows: the result is rounded once; what comes before is fp32, a dozen operations on the addends x cos and x' sin, so
2^-20 of their magnitudes on top.
Attention: the weights p may be rounded to bf16 before the product with V (2^-8 of sum p |v|), the result once more (2^-8 of
itself); scores are fp32 sums of exact products, off by less than 2^-24 * head_dim * |q||k|, which is below 2^-9 here and moves p
by as much: together at most 2^-8 |o| + (2^-8 + 2^-9) sum p |v|."""
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


def tables(n, hd, seed=0):
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(n, hd // 2, generator=g) * 6.28
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)


def filled(n_kv, hd, capacity, elem, window=0, sinks=0, seed=0, layers=1, spread=1.0):
    """A cache with every slot filled, and its K and V in 64 bits [layers, n_kv, capacity, hd]."""
    from nwc_b200 import KVCache
    g = torch.Generator().manual_seed(seed)
    c = KVCache(n_kv, hd, capacity, elem, layers=layers, window=window, sinks=sinks)
    values = []
    for t, e in ((c.k, c.k_exp), (c.v, c.v_exp)):
        x = spread * torch.randn(t.shape, generator=g, dtype=torch.float64)
        if elem == "bf16": t.copy_(x.to(torch.bfloat16)); values.append(x.to(torch.bfloat16).double())
        else:
            u = R.unit_exponent(x)
            codes = R.rounded_e4m3(x * torch.exp2(-u.double())[..., None])
            t.copy_(codes.to(torch.float32).to(torch.float8_e4m3fn)); e.copy_((u + 127).to(torch.uint8))
            values.append(codes * torch.exp2(u.double())[..., None])
    return c, values[0], values[1]


def queries(T, n_q, hd, seed=1, size=1.5):
    return (size * torch.randn(T, n_q, hd, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


def at(pos):
    return torch.tensor([pos], dtype=torch.int32, device="cuda")


def assert_attention(got, want, weight):
    err = (got.double().cpu() - want.reshape(got.shape)).abs()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * weight + 1e-30
    worst = (err / bound.reshape(got.shape)).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, worst


# ---- store and read back ----

@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,hd", [(16, 8, 128), (4, 2, 64), (8, 2, 256), (5, 5, 64), (6, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("T,pos,capacity,window,sinks", [(1, 0, 1, 0, 0), (1, 777, 1024, 0, 0), (37, 5, 42, 0, 0), (53, 90, 117, 64, 1), (3, 1000, 23, 17, 4)])
def test_store_and_read_back(elem, n_q, n_kv, hd, T, pos, capacity, window, sinks):
    from nwc_b200 import KVCache
    g = torch.Generator().manual_seed(T + pos)
    x = 3 * torch.randn(T, (n_q + 2 * n_kv) * hd, generator=g)
    x[:, -hd:] *= torch.exp(4 * torch.randn(T, 1, generator=g))         # rows of very different size
    if T > 2: x[2, -hd:] = 0                                            # a row of zeros
    x = x.to(torch.bfloat16)
    norm = hd != 64
    qn, kn = ((1 + 0.2 * torch.randn(2, hd, generator=g)).to(torch.bfloat16) if norm else (None, None))
    cos, sin = tables(pos + T, hd)
    c = KVCache(n_kv, hd, capacity, elem, layers=2, window=window, sinks=sinks)
    dev = lambda t: None if t is None else t.cuda()
    before = [t.view(torch.uint8).clone() for t in (c.k, c.v)]
    q = c.append(x.cuda(), at(pos), cos.cuda(), sin.cuda(), dev(qn), dev(kn), EPS, layer=1)
    first = max(pos, pos + T - (capacity - sinks)) if window else pos    # what the ring still holds
    k, v = c.read(first, pos + T - first, layer=1)
    c.check()
    heads = x.double().view(T, -1, hd)
    rows = range(pos, pos + T)
    want_q, mag_q = R.turned(heads[:, :n_q], qn, cos[list(rows)], sin[list(rows)], EPS)
    want_k, mag_k = R.turned(heads[:, n_q:n_q + n_kv], kn, cos[list(rows)], sin[list(rows)], EPS)
    want_v = heads[:, n_q + n_kv:]
    assert ((q.double().cpu() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20 * mag_q).all()
    for got, want, mag, exps in ((k, want_k, mag_k, c.k_exp), (v, want_v, want_v.abs() * 0, c.v_exp)):
        got, want, mag = got.double().cpu(), want.transpose(0, 1)[:, first - pos:], mag.transpose(0, 1)[:, first - pos:]
        if elem == "bf16": bound = 2.0 ** -8 * want.abs()
        else:
            slots = torch.tensor([R.slot(p, capacity, window, sinks) for p in range(first, pos + T)])
            unit = torch.exp2(exps[1].cpu()[:, slots].double() - 127)[..., None]
            top = want.abs().amax(-1, keepdim=True)
            assert (top <= 448 * unit * (1 + 2.0 ** -18)).all() and ((top >= 224 * unit * (1 - 2.0 ** -18)) | (top < 1e-36)).all()
            bound = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * unit)
        assert ((got - want).abs() <= bound + 2.0 ** -20 * mag + 1e-40).all()
    if elem == "fp8":                                                    # V goes in as bf16 numbers: its codes are exact
        slots = torch.tensor([R.slot(p, capacity, window, sinks) for p in range(first, pos + T)])
        wv = want_v.transpose(0, 1)[:, first - pos:]
        u = R.unit_exponent(wv)
        assert torch.equal(c.v_exp[1].cpu()[:, slots].int(), (u + 127).int())
        assert torch.equal(R.held(c.v[1].float().cpu()[:, slots], c.v_exp[1].cpu()[:, slots]), R.rounded_e4m3(wv * torch.exp2(-u.double())[..., None]) * torch.exp2(u.double())[..., None])
    assert torch.equal(c.k.view(torch.uint8)[0], before[0][0]) and torch.equal(c.v.view(torch.uint8)[0], before[1][0])      # the other layer is as it was
    touched = {R.slot(p, capacity, window, sinks) for p in rows}
    rest = torch.tensor([s for s in range(capacity) if s not in touched], dtype=torch.long)
    assert torch.equal(c.k.view(torch.uint8)[1].cpu()[:, rest], before[0][1].cpu()[:, rest]) and torch.equal(c.v.view(torch.uint8)[1].cpu()[:, rest], before[1][1].cpu()[:, rest])


def test_store_reads_strided_rows_and_draft_positions():
    from nwc_b200 import KVCache
    n_q, n_kv, hd, T, pos = 8, 2, 128, 9, 30
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(T, (n_q + 2 * n_kv) * hd + 64, generator=g).to(torch.bfloat16).cuda()
    x = wide[:, 32:32 + (n_q + 2 * n_kv) * hd]
    depth = torch.tensor([0, 1, 1, 2, 2, 3, 0, 1, 4], dtype=torch.int32)
    cos, sin = tables(pos + 5, hd)                                       # rows up to the deepest draft's only
    c = KVCache(n_kv, hd, 64, "bf16")
    q = c.append(x, at(pos), cos.cuda(), sin.cuda(), depth=depth.cuda())
    k, v = c.read(pos, T)
    c.check()
    heads, rows = x.cpu().double().reshape(T, -1, hd), pos + depth.long()
    for got, part in ((q, heads[:, :n_q]), (k.transpose(0, 1), heads[:, n_q:n_q + n_kv])):
        want, mag = R.turned(part, None, cos[rows], sin[rows], EPS)
        assert ((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * mag).all()
    assert torch.equal(v.transpose(0, 1).cpu().double(), heads[:, n_q + n_kv:])


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
def test_store_keeps_what_is_not_finite_out_and_reports_it(elem):
    from nwc_b200 import KVCache
    n_q, n_kv, hd = 4, 2, 64
    x = torch.randn(3, (n_q + 2 * n_kv) * hd).to(torch.bfloat16).cuda()
    x[1, n_q * hd + 3] = float("nan"); x[2, -1] = float("inf")
    cos, sin = torch.ones(8, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, hd, dtype=torch.bfloat16, device="cuda")
    c = KVCache(n_kv, hd, 8, elem)
    c.append(x, at(2), cos, sin)
    k, v = c.read(2, 3)
    assert torch.isfinite(k).all() and torch.isfinite(v).all() and k[0, 1, 3] == 0 and v[1, 2, -1] == 0 and k[0, 1, 4] != 0
    with pytest.raises(RuntimeError, match="finite"): c.check()
    c.check()                                                            # reported once


def test_largest_and_smallest_rows_survive_quantising():
    from nwc_b200 import KVCache
    hd = 64
    rows = torch.zeros(6, hd)
    rows[0, 0], rows[1, 0], rows[2, 0], rows[3, 5], rows[4, :] = 3.3895313892515355e38, 448.0, 450.0, 1e-38, 2.0 ** -130
    x = torch.zeros(6, 3 * hd); x[:, 2 * hd:] = rows
    x = x.to(torch.bfloat16)
    one, zero = torch.ones(6, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, hd, dtype=torch.bfloat16, device="cuda")
    c = KVCache(1, hd, 6, "fp8")
    c.append(x.cuda(), at(0), one, zero)
    _, v = c.read(0, 6)
    c.check()
    want = x[:, 2 * hd:].double()
    unit = torch.exp2(c.v_exp[0, 0].cpu().double() - 127)[:, None]
    assert ((v[0].double().cpu() - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * unit)).all()
    assert c.v_exp[0, 0].cpu().tolist()[1:3] == [127, 128] and int(c.v_exp[0, 0, 5]) == 0 and (v[0, 5] == 0).all()


def test_read_back_of_every_code():
    """All 256 codes under several exponents, the NaN codes among them: exactly code * 2^(b - 127), rounded to bf16 once where
    that is below bf16's normal range."""
    from nwc_b200 import KVCache
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 4, 64).repeat(1, 1, 6, 1).cuda()
    exps = torch.tensor([0, 1, 9, 127, 200, 246], dtype=torch.uint8).repeat_interleave(4).view(1, 1, 24).cuda()
    c = KVCache.over(codes.view(torch.float8_e4m3fn).contiguous(), codes.view(torch.float8_e4m3fn).clone(), exps, exps.clone())
    k, v = c.read(0, 24)
    want = (codes.view(torch.float8_e4m3fn).float().cpu().double() * torch.exp2(exps.cpu().double() - 127)[..., None])[0]
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(k.cpu()), nan) and torch.equal(torch.isnan(v.cpu()), nan)
    assert torch.equal(k.cpu().double()[~nan], want.to(torch.bfloat16).double()[~nan]) and torch.equal(k.cpu()[~nan], v.cpu()[~nan])


# ---- attention ----

SHAPES = [(16, 8, 128), (4, 2, 64), (8, 1, 128), (6, 2, 128), (5, 5, 64), (8, 2, 256)]


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,hd", SHAPES)
@pytest.mark.parametrize("T,pos,spare", [(1, 0, 0), (1, 1, 3), (1, 127, 0), (1, 128, 900), (1, 700, 1), (2, 0, 0), (5, 254, 0), (33, 100, 7), (130, 0, 0), (129, 300, 0)])
def test_attention_over_everything(elem, n_q, n_kv, hd, T, pos, spare):
    c, k, v = filled(n_kv, hd, pos + T + spare, elem, seed=pos + T)
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos))


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,hd", [(16, 8, 128), (4, 2, 64), (8, 2, 256)])
@pytest.mark.parametrize("T,pos,window,sinks,spare", [(1, 0, 1, 0, 0), (1, 5, 1, 0, 0), (1, 5, 1, 3, 0), (1, 40, 64, 4, 0), (1, 5000, 300, 4, 0), (1, 777, 128, 0, 5), (1, 900, 200, 130, 3),
                                                      (7, 1000, 100, 4, 0), (40, 10, 16, 4, 0), (150, 0, 33, 2, 0), (140, 2000, 257, 7, 11), (130, 60, 500, 1, 0)])
def test_attention_with_a_window_and_sinks(elem, n_q, n_kv, hd, T, pos, window, sinks, spare):
    c, k, v = filled(n_kv, hd, sinks + window + T - 1 + spare, elem, window, sinks, seed=pos + T)
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos, window, sinks))


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("n_q,n_kv,hd", [(16, 8, 128), (4, 2, 64), (8, 2, 256), (8, 1, 128)])
@pytest.mark.parametrize("T,pos,window,sinks", [(1, 0, 0, 0), (2, 50, 0, 0), (26, 120, 0, 0), (33, 0, 0, 0), (64, 700, 0, 0), (48, 3000, 200, 4), (65, 5, 40, 2), (140, 250, 0, 0)])
def test_attention_of_a_draft_tree(elem, n_q, n_kv, hd, T, pos, window, sinks):
    from nwc_b200 import draft_tree
    g = torch.Generator().manual_seed(T)
    parents = [-1] + [int(torch.randint(-1 if i % 9 == 0 else max(0, i - 7), i, (1,), generator=g)) for i in range(1, T)]
    visible, depth = draft_tree(parents)
    c, k, v = filled(n_kv, hd, sinks + window + T - 1 if window else pos + T, elem, window, sinks, seed=pos + T)
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos), visible=visible, depth=depth)
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos, window, sinks, visible.cpu(), depth.cpu()))


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("T,pos,window,sinks", [(12, 300, 8, 0), (12, 1, 5, 4), (70, 2000, 33, 3), (6, 9000, 1, 2)])
def test_a_chain_of_drafts_longer_than_the_window(elem, T, pos, window, sinks):
    """As a chain, a chunk sees what it sees as a chunk."""
    from nwc_b200 import draft_tree
    n_q, n_kv, hd = 8, 2, 128
    c, k, v = filled(n_kv, hd, sinks + window + T - 1, elem, window, sinks, seed=T)
    q = queries(T, n_q, hd)
    visible, depth = draft_tree([t - 1 for t in range(T)], window=window, sinks=sinks, pos=pos)
    out = c.attend(q.cuda(), at(pos), visible=visible, depth=depth)
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos, window, sinks))


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("T,pos", [(5, 0), (70, 0), (5, 40), (70, 300)])
def test_drafts_that_see_nothing_or_not_themselves(elem, T, pos):
    """Masks other than a tree's: empty rows give zeros where nothing is cached, bits beyond a token's own position count."""
    n_q, n_kv, hd = 8, 2, 128
    rows = [[] if t % 3 == 0 else [T - 1 - t] if t % 3 == 1 else list(range(T)) for t in range(T)]
    visible, depth = R.tree_bits(T, rows), torch.zeros(T, dtype=torch.int32)
    c, k, v = filled(n_kv, hd, pos + T, elem, seed=T)
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos), visible=visible.cuda(), depth=depth.cuda())
    c.check()
    want, weight = R.attend(q.double(), k[0], v[0], pos, visible=visible, depth=depth)
    assert_attention(out, want, weight)
    if pos == 0: assert (out[0::3] == 0).all()


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("elem", ["bf16", "fp8"])
def test_what_lies_outside_the_visible_span_does_not_matter(elem, T):
    """NaN and infinities in slots that no token of the call sees: behind the last token, in front of the window."""
    n_q, n_kv, hd, pos, window, sinks = 8, 2, 128, 1000, 150, 3
    c, k, v = filled(n_kv, hd, 700, elem, window, sinks, seed=T)
    seen = {R.slot(p, 700, window, sinks) for p in range(pos + T) if p < sinks or p > pos - window}
    out_of_sight = torch.tensor([s for s in range(700) if s not in seen])
    for t in (c.k, c.v):
        raw = t.view(torch.uint8) if elem == "fp8" else t
        raw[:, :, out_of_sight.cuda()] = 0x7F if elem == "fp8" else float("nan")
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos, window, sinks))


@pytest.mark.parametrize("T,n_q,n_kv,hd", [(1300, 128, 8, 64), (1199, 128, 8, 64), (650, 128, 4, 64), (1215, 16, 1, 64), (5200, 8, 1, 64)])
def test_more_row_tiles_than_the_gpu_has_places(T, n_q, n_kv, hd):
    """Waves of units whose last one is halved (whole, with an odd tile, with few rows left), or is not; against torch in fp32
    here, its error (2^-20) being no part of the bound."""
    pos, window, sinks = 100, 70, 3
    c, k, v = filled(n_kv, hd, sinks + window + T - 1, "bf16", window, sinks, seed=T)
    q = queries(T, n_q, hd).cuda()
    out = c.attend(q, at(pos)).view(T, n_q, hd)
    c.check()
    k, v = k[0].float().cuda(), v[0].float().cuda()
    p = torch.tensor([x for x in range(pos + T) if x < sinks or x > pos - window], device="cuda")
    slots = torch.tensor([R.slot(int(x), sinks + window + T - 1, window, sinks) for x in p], device="cuda")
    own = pos + torch.arange(T, device="cuda")[:, None]
    sees = (p <= own) & ((p < sinks) | (p > own - window))
    for h in range(0, n_q, max(1, n_q // 16)):
        g = h // (n_q // n_kv)
        w = torch.softmax((q[:, h].float() @ k[g, slots].T / hd ** 0.5).masked_fill(~sees, float("-inf")), -1)
        assert_attention(out[:, h], (w @ v[g, slots]).double().cpu(), (w @ v[g, slots].abs()).double().cpu())


@pytest.mark.parametrize("T", [1, 40, 200])
def test_scores_of_any_size(T):
    """Score differences of hundreds (one position takes all the weight) and a scale of the caller's; scores that large stay
    within the bound because it is relative to sum p |v|, p being 0 or 1."""
    n_q, n_kv, hd, pos = 4, 2, 64, 333
    c, k, v = filled(n_kv, hd, pos + T, "bf16", seed=T, spread=4.0)
    q = queries(T, n_q, hd, size=64.0)
    out = c.attend(q.cuda(), at(pos), scale=0.5)
    c.check()
    assert_attention(out, *R.attend(q.double(), k[0], v[0], pos, scale=0.5))


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_value_rows_of_very_different_size(T, hd):
    """Every second position holds values 2^-22 of its neighbours'; the keys make queries prefer the small ones so clearly
    (scores 60 apart) that the large ones weigh nothing: the small values come out to the usual precision."""
    from nwc_b200 import KVCache
    n_q, n_kv, pos = 8, 2, 300
    g = torch.Generator().manual_seed(T)
    c = KVCache(n_kv, hd, pos + T, "fp8")
    small = torch.arange(pos + T) % 2 == 1
    k = torch.randn(n_kv, pos + T, hd, generator=g, dtype=torch.float64) * 0.1
    k[:, small, 0] += 8.0; k[:, ~small, 0] -= 8.0
    v = torch.randn(n_kv, pos + T, hd, generator=g, dtype=torch.float64) * torch.where(small, 2.0 ** -22, 1.0)[:, None].double()
    held = []
    for x, t, e in ((k, c.k, c.k_exp), (v, c.v, c.v_exp)):
        u = R.unit_exponent(x)
        codes = R.rounded_e4m3(x * torch.exp2(-u.double())[..., None])
        t[0].copy_(codes.to(torch.float32).to(torch.float8_e4m3fn)); e[0].copy_((u + 127).to(torch.uint8))
        held.append(codes * torch.exp2(u.double())[..., None])
    q = torch.randn(T, n_q, hd, generator=g) * 0.1
    q[:, :, 0] = 4.0 * hd ** 0.5
    q = q.to(torch.bfloat16)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    want, weight = R.attend(q.double(), held[0], held[1], pos)
    assert want.abs().max() < 2.0 ** -18
    assert_attention(out, want, weight)


def quantised_into(c, k, v):
    """64-bit rows k, v [n_kv, positions, hd] into the first slots of an fp8 cache; what it then holds."""
    held = []
    for x, t, e in ((k, c.k, c.k_exp), (v, c.v, c.v_exp)):
        u = R.unit_exponent(x)
        codes = R.rounded_e4m3(x * torch.exp2(-u.double())[..., None])
        n = x.shape[1]
        t.view(torch.uint8)[0, :, :n] = codes.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
        e[0, :, :n] = (u + 127).to(torch.uint8).cuda()
        held.append(codes * torch.exp2(u.double())[..., None])
    return held


@pytest.mark.parametrize("bits,ratio", [(12, 6), (12, 10), (16, 6), (16, 10), (20, 6), (20, 10), (28, 9), (40, 0)])
@pytest.mark.parametrize("hd,T,positions,first", [(128, 1, 700, "zero"), (128, 1, 9000, "zero"), (64, 5, 9000, "zero"), (256, 1, 6000, "zero"), (128, 3, 5000, "small"), (256, 1, 30000, "like the others")])
def test_a_first_token_that_takes_almost_all_the_weight(bits, ratio, hd, T, positions, first):
    """A sink: every other key's weight is 2^-bits of the first one's, whose value is zero, small or large; values are 2^-ratio of
    one outlier's.  What the small weights bring comes out to the usual precision (there is no other output where the first value is zero)."""
    from nwc_b200 import KVCache
    n_q, n_kv, pos = 8, 2, positions - T
    g = torch.Generator().manual_seed(bits + hd)
    c = KVCache(n_kv, hd, positions, "fp8")
    k = 0.1 * torch.randn(n_kv, positions, hd, generator=g, dtype=torch.float64)
    v = torch.randn(n_kv, positions, hd, generator=g, dtype=torch.float64) * 2.0 ** -ratio
    k[:, :, 0] = 0.0; k[:, 0, 0] = 8.0
    v[:, 37] *= 2.0 ** ratio
    v[:, 0] *= {"zero": 0.0, "small": 1.0, "like the others": 2.0 ** ratio}[first]
    held = quantised_into(c, k, v)
    q = torch.randn(T, n_q, hd, generator=g) * 0.1
    q[:, :, 0] = bits * 0.6931 * hd ** 0.5 / 8.0
    q = q.to(torch.bfloat16)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    assert_attention(out, *R.attend(q.double(), *held, pos))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("positions,capacity", [(3, 3), (700, 700), (700, 6000)])
def test_a_large_value_of_little_weight_beside_small_values(hd, positions, capacity):
    """One value 2^28 of the others', with a weight of 2^-12 and zeros in half of its dimensions: in those, what the others bring
    comes out to the usual precision."""
    from nwc_b200 import KVCache
    n_q, n_kv, pos = 8, 2, positions - 1
    g = torch.Generator().manual_seed(hd + positions)
    c = KVCache(n_kv, hd, capacity, "fp8")
    k = 0.1 * torch.randn(n_kv, positions, hd, generator=g, dtype=torch.float64)
    k[:, :, 0] = 8.0; k[:, 1, 0] = 0.0
    v = torch.randn(n_kv, positions, hd, generator=g, dtype=torch.float64) * 2.0 ** -28
    v[:, 1] *= 2.0 ** 28; v[:, 1, ::2] = 0.0
    held = quantised_into(c, k, v)
    q = torch.randn(1, n_q, hd, generator=g) * 0.1
    q[:, :, 0] = 12 * 0.6931 * hd ** 0.5 / 8.0
    q = q.to(torch.bfloat16)
    out = c.attend(q.cuda(), at(pos))
    c.check()
    assert_attention(out, *R.attend(q.double(), *held, pos))


@pytest.mark.parametrize("hd,T,n_q,larger", [(256, 6, 16, 135), (128, 2, 8, 100), (64, 2, 8, 100)])
def test_values_that_a_row_does_not_see_do_not_cost_it_precision(hd, T, n_q, larger):
    """The last token's value is 2^100 of the others' (2^135 where its rows are computed apart from theirs): the tokens in front
    of it are as precise as ever.  Compared times 2^60."""
    from nwc_b200 import KVCache
    n_kv, pos = 1, 500
    g = torch.Generator().manual_seed(hd)
    c = KVCache(n_kv, hd, 5000, "fp8")
    k = 0.3 * torch.randn(n_kv, pos + T, hd, generator=g, dtype=torch.float64)
    v = torch.randn(n_kv, pos + T, hd, generator=g, dtype=torch.float64) * 2.0 ** -60
    v[:, -1] *= 2.0 ** larger
    held = quantised_into(c, k, v)
    q = queries(T, n_q, hd)
    out = c.attend(q.cuda(), at(pos)).view(T, n_q, hd)
    c.check()
    want, weight = R.attend(q.double(), *held, pos)
    assert_attention(out[:-1].double() * 2.0 ** 60, want[:-1] * 2.0 ** 60, weight[:-1] * 2.0 ** 60)
    assert_attention(out[-1:], want[-1:], weight[-1:])


def test_query_rows_may_be_slices():
    n_q, n_kv, hd, pos, T = 8, 2, 128, 90, 20
    c, k, v = filled(n_kv, hd, pos + T, "fp8")
    wide = queries(T, n_q + 3, hd).cuda()
    q = wide[:, :n_q]
    out = c.attend(q, at(pos))
    c.check()
    assert_attention(out, *R.attend(q.cpu().double(), k[0], v[0], pos))


def test_strides_of_single_rows_and_heads_do_not_matter():
    """Torch gives a dimension of one any stride."""
    hd, pos = 128, 40
    c, k, v = filled(1, hd, 64, "bf16")
    qkv = queries(1, 3, hd).reshape(1, 3 * hd).cuda()
    cos, sin = (t.cuda() for t in tables(64, hd))
    want = c.append(qkv, at(pos), cos, sin)
    for stride in (1, 4):
        assert torch.equal(c.append(qkv.as_strided((1, 3 * hd), (stride, 1)), at(pos), cos, sin), want)
        assert torch.equal(c.attend(want.as_strided((1, 1, hd), (stride, stride, 1)), at(pos)), c.attend(want, at(pos)))
    q = queries(5, 1, hd).cuda()
    assert torch.equal(c.attend(q.as_strided((5, 1, hd), (hd, 1, 1)), at(pos)), c.attend(q, at(pos)))
    c.check()


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
def test_offsets_beyond_32_bits(elem):
    """Layers whose bytes lie beyond 2^32 of the cache's first."""
    from nwc_b200 import KVCache
    n_q, n_kv, hd, capacity, layers, T, pos = 4, 2, 256, 1 << 19, 17 if elem == "fp8" else 9, 3, (1 << 19) - 3
    c = KVCache(n_kv, hd, capacity, elem, layers=layers)
    assert (layers - 1) * n_kv * capacity * hd * (1 if elem == "fp8" else 2) >= 1 << 32
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, (n_q + 2 * n_kv) * hd, generator=g).to(torch.bfloat16).cuda()
    one, zero = torch.ones(capacity, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(capacity, hd, dtype=torch.bfloat16, device="cuda")
    q = c.append(x, at(pos), one, zero, layer=layers - 1)
    k, v = c.read(pos, T, layer=layers - 1)
    if elem == "bf16": assert torch.equal(v.transpose(0, 1).reshape(T, -1), x[:, (n_q + n_kv) * hd:])
    visible, depth = R.tree_bits(T, [[0], [0, 1], [2]]), torch.zeros(T, dtype=torch.int32)
    out = c.attend(q, at(pos), visible=visible.cuda(), depth=depth.cuda(), layer=layers - 1)
    c.check()
    # the cached part: zero keys (score 0) and zero values, pos of them
    want, weight = torch.zeros(T, n_q, hd, dtype=torch.float64), torch.zeros(T, n_q, hd, dtype=torch.float64)
    for t, seen in enumerate([[0], [0, 1], [2]]):
        for h in range(n_q):
            x_ = torch.exp((k[h // 2, seen].cpu().double() @ q[t, h].cpu().double()) / hd ** 0.5)
            want[t, h] = (x_ @ v[h // 2, seen].cpu().double()) / (x_.sum() + pos)
            weight[t, h] = (x_ @ v[h // 2, seen].cpu().double().abs()) / (x_.sum() + pos)
    # sums of half a million equal weights: fp32 running sums of at most 2^19 terms are exact to 2^-24 * 2^5 when added in pieces, 2^-8 covers them
    err = (out.cpu().double().view(T, n_q, hd) - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -6 * weight).all()


@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 2, 256), (256, 8, 64)])
def test_the_most_tokens_of_a_call(n_q, n_kv, hd):
    """65535 tokens of so many heads that the row tiles pass 65535, each seeing itself alone: its value comes back."""
    from nwc_b200 import KVCache
    T = 65535
    c = KVCache(n_kv, hd, T, "bf16", window=1)
    c.v.copy_(torch.randn(c.v.shape[2:], device="cuda").to(torch.bfloat16)[None, None].expand_as(c.v))
    q = torch.ones(T, n_q, hd, dtype=torch.bfloat16, device="cuda")
    out = c.attend(q, at(7)).view(T, n_q, hd)
    c.check()
    slots = (7 + torch.arange(T, device="cuda")) % T
    assert torch.equal(out, c.v[0, 0][slots][:, None].expand_as(out))


@pytest.mark.parametrize("T,pos", [(1, 200), (60, 200), (1, 9000), (5, 9000), (300, 700)])
def test_queries_that_are_not_finite_spoil_their_own_rows_only(T, pos):
    n_q, n_kv, hd = 8, 2, 128
    c, k, v = filled(n_kv, hd, pos + T, "fp8")
    q = queries(T, n_q, hd)
    q[0, 3, 5] = float("nan")
    out = c.attend(q.cuda(), at(pos)).view(T, n_q, hd)
    c.check()
    assert torch.isnan(out[0, 3]).all()
    keep = torch.ones(T, n_q, dtype=torch.bool); keep[0, 3] = False
    q[0, 3] = 0
    want, weight = R.attend(q.double(), k[0], v[0], pos)
    assert_attention(out[keep.cuda()], want[keep], weight[keep])


def test_calls_on_other_streams_and_from_two_caches():
    """A call's workspace is its own: two caches attended from two streams at the same time, many times."""
    n_q, n_kv, hd, pos = 16, 2, 128, 6000
    made = [filled(n_kv, hd, pos + 64, "fp8", seed=s) for s in (1, 2)]
    qs = [queries(T, n_q, hd, seed=T).cuda() for T in (1, 40)]
    p = at(pos)
    want = [[c.attend(q, p) for q in qs] for c, _, _ in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s): got[i].append([made[i][0].attend(q, p) for q in qs])
    torch.cuda.synchronize()
    for i in (0, 1):
        made[i][0].check()
        for outs in got[i]: assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


# ---- the operators together ----

@pytest.mark.parametrize("elem", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_a_session_of_chunks_drafts_and_tokens(elem, window, sinks):
    """A prompt in two chunks, a draft tree, the accepted path moved together, then single tokens: every output agrees with a
    64-bit attention over what the cache holds, and the moved rows are the drafts' rows bit for bit."""
    from nwc_b200 import KVCache, draft_tree
    n_q, n_kv, hd, total = 8, 2, 128, 260
    capacity = sinks + window + 100 if window else total
    g = torch.Generator().manual_seed(11)
    cos, sin = tables(total, hd)
    cos_d, sin_d = cos.cuda(), sin.cuda()
    c = KVCache(n_kv, hd, capacity, elem, layers=2, window=window, sinks=sinks)
    position = torch.zeros(1, dtype=torch.int32, device="cuda")
    fresh = lambda T: torch.randn(T, (n_q + 2 * n_kv) * hd, generator=g).to(torch.bfloat16).cuda()
    def values():
        if elem == "bf16": return c.k[1].cpu().double(), c.v[1].cpu().double()
        return R.held(c.k[1].float().cpu(), c.k_exp[1].cpu()), R.held(c.v[1].float().cpu(), c.v_exp[1].cpu())
    def go(T, visible=None, depth=None):
        q = c.append(fresh(T), position, cos_d, sin_d, depth=depth, layer=1)
        out = c.attend(q, position, visible=visible, depth=depth, layer=1)
        k, v = values()
        on_cpu = lambda t: None if t is None else t.cpu()
        assert_attention(out, *R.attend(q.cpu().double(), k, v, int(position), window, sinks, on_cpu(visible), on_cpu(depth)))
    for T in (97, 61): go(T); position += T
    parents = [-1, 0, 0, 1, 2, 2, 4, 4, 7, -1, 9]
    visible, depth = draft_tree(parents)
    go(len(parents), visible, depth)
    drafts = c.read(int(position), len(parents), layer=1)
    path, count = torch.tensor([0, 2, 4, 7, 8, 10], dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    c.commit(position, path, count, tokens=len(parents))
    moved = c.read(int(position), len(parents), layer=1)
    for a, b in zip(drafts, moved):
        assert torch.equal(b[:, :5], a[:, [0, 2, 4, 7, 8]]) and torch.equal(b[:, 5:], a[:, 5:])
    position += count
    for _ in range(3): go(1); position += 1
    c.check()


def test_the_first_layer_is_not_moved_by_another_caches_commit_and_all_layers_are():
    from nwc_b200 import KVCache
    c = KVCache(2, 64, 32, "fp8", layers=3)
    raw = [c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_exp, c.v_exp]
    for i, t in enumerate(raw): t.copy_(torch.randint(0, 120, t.shape, generator=torch.Generator().manual_seed(i), dtype=torch.uint8))
    was = [t.clone() for t in raw]
    c.commit(at(10), torch.tensor([1, 3, 4], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"), tokens=6)
    c.check()
    for t, w in zip(raw, was):
        w[:, :, 10:13] = w[:, :, [11, 13, 14]]
        assert torch.equal(t, w)


@pytest.mark.parametrize("window,sinks,capacity,pos", [(0, 0, 40, 33), (0, 0, 40, 0), (20, 3, 30, 33), (20, 3, 30, 1000)])
def test_commit_finds_the_trees_limits_itself(window, sinks, capacity, pos):
    c, k, v = filled(2, 64, capacity, "fp8", window, sinks)
    was = c.read(pos, 7)
    path = [0, 2, 3, 6]
    c.commit(at(pos), torch.tensor(path, dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda"))
    c.check()
    for a, b in zip(was, c.read(pos, 7)): assert torch.equal(b[:, :4], a[:, path]) and torch.equal(b[:, 4:], a[:, 4:])
    beyond = 40 - pos if not window else 8                              # the first draft that the cache could not have taken
    c.commit(at(pos), torch.tensor([beyond], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="path"): c.check()


@pytest.mark.parametrize("path,count,tokens", [([2, 1], 2, 4), ([0, 0], 2, 4), ([0, 4], 2, 4), ([-1, 0], 2, 4), ([0, 1], 3, 4), ([0, 1], -1, 4)])
def test_wrong_paths_move_nothing(path, count, tokens):
    c, _, _ = filled(2, 64, 32, "bf16")
    was = c.k.clone()
    c.commit(at(10), torch.tensor(path, dtype=torch.int32, device="cuda"), torch.tensor([count], dtype=torch.int32, device="cuda"), tokens=tokens)
    with pytest.raises(RuntimeError, match="path"): c.check()
    assert torch.equal(c.k, was)


@pytest.mark.parametrize("pos,window", [(30, 0), (-1, 0), (-1, 16), (2 ** 31 - 2, 16)])
def test_positions_outside_the_cache_write_nothing(pos, window):
    c, _, _ = filled(2, 64, 32, "bf16", window, 4 if window else 0)
    was = c.k.clone()
    x = torch.randn(3, 8 * 64).to(torch.bfloat16).cuda()
    cos = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda")
    c.append(x, at(pos), cos, cos)
    with pytest.raises(RuntimeError, match="position"): c.check()
    c.attend(x.view(3, 8, 64), at(pos))
    with pytest.raises(RuntimeError, match="position"): c.check()
    assert torch.equal(c.k, was)


def test_rotary_rows_beyond_the_tables_write_nothing():
    c, _, _ = filled(2, 64, 32, "bf16")
    was = c.k.clone()
    x = torch.randn(3, 8 * 64).to(torch.bfloat16).cuda()
    cos = torch.ones(12, 64, dtype=torch.bfloat16, device="cuda")
    c.append(x, at(10), cos, cos)
    with pytest.raises(RuntimeError, match="position"): c.check()
    assert torch.equal(c.k, was)
    c.append(x, at(10), cos, cos, depth=torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))       # the third draft's row is missing
    with pytest.raises(RuntimeError, match="position"): c.check()
    assert torch.equal(c.k[:, :, 12], was[:, :, 12]) and not torch.equal(c.k[:, :, 10], was[:, :, 10])


@pytest.mark.parametrize("T", [1, 9, 150])
def test_captured_and_replayed_calls_follow_the_position(T):
    """A step captured once is replayed at other positions; two graphs replayed on two streams do not disturb each other."""
    n_q, n_kv, hd, capacity = 8, 2, 128, 600
    made = [filled(n_kv, hd, capacity, "fp8", seed=s) for s in (1, 2)]
    x = [torch.randn(T, (n_q + 2 * n_kv) * hd, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).cuda() for s in (3, 4)]
    cos, sin = (t.cuda() for t in tables(capacity, hd))
    where, graphs, outs = [at(5), at(5)], [], []
    for (c, _, _), xi, p in zip(made, x, where):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side): c.attend(c.append(xi, p, cos, sin), p)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g): outs.append(c.attend(c.append(xi, p, cos, sin), p))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for pos in (0, 17, 440):
        for p in where: p.fill_(pos)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s): g.replay()
        torch.cuda.synchronize()
        for (c, _, _), xi, p, out in zip(made, x, where, outs):
            got = out.clone()
            want = c.attend(c.append(xi, p, cos, sin), p)
            c.check()
            assert torch.equal(got, want)


def test_what_the_python_calls_refuse():
    from nwc_b200 import KVCache
    c = KVCache(2, 64, 32, "fp8", layers=2)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    x, p, t, w = bf(3, 8 * 64), at(0), bf(40, 64), bf(64)
    good = dict(qkv=x, pos=p, cos=t, sin=t, q_norm=w, k_norm=w)
    for bad in (dict(qkv=x.float()), dict(qkv=x.cpu()), dict(qkv=bf(3, 8 * 64 + 1)), dict(qkv=bf(3, 3 * 64)), dict(qkv=bf(3, 7 * 64)), dict(qkv=bf(8 * 64, 3).T), dict(qkv=bf(0, 8 * 64)),
                dict(pos=torch.zeros(1, device="cuda")), dict(pos=p.cpu()), dict(pos=p.repeat(2)), dict(cos=t[:, :32]), dict(cos=t.float()), dict(cos=bf(39, 64)), dict(sin=bf(64, 40).T),
                dict(q_norm=None), dict(k_norm=w[:32]), dict(q_norm=w.float()), dict(depth=p), dict(depth=torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError): c.append(**{**good, **bad})
    for layer in (-1, 2):
        with pytest.raises(IndexError): c.append(**good, layer=layer)
        with pytest.raises(IndexError): c.read(0, 1, layer=layer)
    q, words = bf(3, 4, 64), torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    good = dict(q=q, pos=p)
    for bad in (dict(q=q.float()), dict(q=bf(3, 5, 64)), dict(q=bf(3, 4, 128)), dict(q=bf(3, 4 * 64)), dict(q=bf(4, 3, 64).transpose(0, 1)), dict(visible=words), dict(depth=p),
                dict(visible=words, depth=p), dict(visible=words[:2], depth=words.view(3)), dict(scale=0.0), dict(scale=float("nan")), dict(q=bf(33, 4, 64))):
        with pytest.raises(ValueError): c.attend(**{**good, **bad})
    with pytest.raises(IndexError): c.attend(q, p, layer=5)
    for first, count in ((-1, 2), (0, 0), (30, 3)):
        with pytest.raises(ValueError): c.read(first, count)
    for path, count in ((torch.zeros(2, 1, dtype=torch.int32, device="cuda"), p), (p.float(), p), (p, p.cpu())):
        with pytest.raises(ValueError): c.commit(p, path, count)
    ring = KVCache(2, 64, 32, window=20, sinks=2)
    with pytest.raises(ValueError): ring.append(bf(12, 8 * 64), p, t, t)                # 30 slots hold a window of 20 and 11 tokens, not 12
    ring.append(bf(11, 8 * 64), p, t, t)
    with pytest.raises(ValueError): ring.read(2, 31)
    c.append(**dict(qkv=x[0], pos=p, cos=t, sin=t))                                     # a vector is one token
    c.check(); ring.check()


def test_a_wait_that_ran_out_is_reported_by_the_cache_and_by_the_library():
    """The probe waits, for a moment, for a barrier that nothing arrives at, and reports it as the attention kernel does."""
    from nwc_b200 import KVCache, _lib as L
    c = KVCache(2, 64, 32)
    assert L.lib.nwc_kernel_status(1) == 0
    assert L.lib.nwc_kv_wait_probe(L.stream(), L.ptr(c.status)) == 0
    with pytest.raises(RuntimeError, match="gave up"): c.check()
    c.check()                                                            # reported once
    assert L.lib.nwc_kernel_status(0) == 2 and L.lib.nwc_kernel_status(1) == 2 and L.lib.nwc_kernel_status(1) == 0


def test_gradients_are_not_lost_silently():
    c, _, _ = filled(2, 64, 32, "bf16")
    qkv, t, w = queries(3, 8, 64).reshape(3, 512).cuda(), torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q = c.append(qkv, at(0), t, t, w, w)
    wants = lambda x: x.clone().requires_grad_()
    for call in (lambda: c.append(wants(qkv), at(0), t, t, w, w), lambda: c.append(qkv, at(0), t, t, wants(w), w), lambda: c.append(qkv, at(0), t, t, w, wants(w)), lambda: c.attend(wants(q), at(0))):
        with pytest.raises(ValueError, match="no_grad"): call()
    with torch.no_grad(): assert torch.equal(c.append(wants(qkv), at(0), t, t, wants(w), w), q) and torch.equal(c.attend(wants(q), at(0)), c.attend(q, at(0)))
    c.check()


@pytest.mark.parametrize("elem,window,sinks", [("bf16", 0, 0), ("fp8", 40, 4)])
def test_a_captured_verification_follows_position_path_and_count(elem, window, sinks):
    """Store, attention and commit of a draft tree in one graph, replayed with other positions, paths and counts on the device."""
    from nwc_b200 import draft_tree
    n_q, n_kv, hd, T = 8, 2, 128, 9
    capacity = sinks + window + T - 1 if window else 300
    made = [filled(n_kv, hd, capacity, elem, window, sinks, seed=5, layers=2)[0] for _ in range(2)]
    cos, sin = (t.cuda() for t in tables(700, hd))
    x = torch.randn(T, (n_q + 2 * n_kv) * hd, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    visible, depth = draft_tree([-1, 0, 0, 1, 2, 2, 4, 4, 7], window=window, sinks=sinks, pos=100)
    p, path, count = at(100), torch.zeros(T, dtype=torch.int32, device="cuda"), at(0)
    def step(c):
        q = c.append(x, p, cos, sin, depth=depth, layer=1)
        out = c.attend(q, p, visible=visible, depth=depth, layer=1)
        c.commit(p, path, count, tokens=T)
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side): step(made[0]); step(made[1])
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g): out = step(made[0])
    bits = lambda c: [t.view(torch.uint8) for t in (c.k, c.v, c.k_exp, c.v_exp) if t is not None]
    for pos, way in ((100, [0, 2, 5]), (103, [0, 1, 3]), (250, [0, 2, 4, 7, 8]), (251, [0])):
        p.fill_(pos); path[:len(way)] = torch.tensor(way, dtype=torch.int32, device="cuda"); count.fill_(len(way))
        g.replay()
        want = step(made[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(bits(made[0]), bits(made[1])): assert torch.equal(a, b)
    for c in made: c.check()


@pytest.mark.parametrize("elem", ["bf16", "fp8"])
def test_the_most_tokens_stored_at_once(elem):
    from nwc_b200 import KVCache
    T, n_q, n_kv, hd = 65535, 3, 1, 64
    c = KVCache(n_kv, hd, T + 5, elem)
    x = torch.randn(T, (n_q + 2 * n_kv) * hd, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    one, zero = torch.ones(T + 5, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(T + 5, hd, dtype=torch.bfloat16, device="cuda")
    q = c.append(x, at(5), one, zero)
    k, v = c.read(5, T)
    c.check()
    assert torch.equal(q.view(T, -1), x[:, :n_q * hd])
    for got, want, byte in ((k[0], x[:, n_q * hd:(n_q + 1) * hd], c.k_exp), (v[0], x[:, (n_q + 1) * hd:], c.v_exp)):
        if elem == "bf16": assert torch.equal(got, want); continue
        u = R.unit_exponent(want.cpu())                                  # (what is stored is a bf16 number: its code is exact)
        assert torch.equal(byte[0, 0, 5:].cpu().int(), (u + 127).int())
        assert torch.equal(got.cpu().double(), R.rounded_e4m3(want.cpu().double() * torch.exp2(-u.double())[:, None]) * torch.exp2(u.double())[:, None])
