"""The decode loop on a KVCache (quantised, under a window, several tokens at once).  What is compared: logits, against the same
engine's plain arrays where both hold the same thing, and against a 64-bit restatement of one layer's attention where they do
not; tokens only where the engine's own two ways of computing the same thing are compared, up to near-ties of the two best logits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def engine(layout=2, max_len=128, layers=2, **kw):
    from nwc_b200.decode import DecodeEngine, DecoderConfig, DecoderWeights
    cfg = DecoderConfig("tiny", layers, 256, 1000, 4, 2, 64, 2048, True, True)
    return DecodeEngine(DecoderWeights.synthetic(cfg, layout=layout, seed=3), max_len=max_len, **kw)


def logits_after(eng, tokens):
    eng.reset()
    out = []
    for t in tokens:
        eng.cur.fill_(t); eng.forward_token(); out.append(eng.logits.float().clone())
    eng._check_status()
    return torch.stack(out)


# Every activation of the loop is rounded to bf16 (2^-8), about ten times per layer, in both engines and after different sums:
# with two layers the logits agree to a few parts in a hundred of their size; 0.1 of the largest leaves room for it, and a wrong
# position, mask or row is off by the size of the logits themselves.
def assert_close(a, b, share=0.1):
    assert torch.isfinite(a).all() and (a - b).abs().max() <= share * b.abs().max(), ((a - b).abs().max() / b.abs().max()).item()


TOKENS = [int(t) for t in torch.randint(0, 2048, (40,), generator=torch.Generator().manual_seed(2))]


@pytest.mark.parametrize("layout", [0, 2])
def test_bf16_cache_agrees_with_the_plain_arrays(layout):
    assert_close(logits_after(engine(layout, chunk=8), TOKENS), logits_after(engine(layout), TOKENS))


def test_a_window_longer_than_the_text_changes_nothing():
    a, b = logits_after(engine(chunk=8), TOKENS), logits_after(engine(window=64, sinks=4), TOKENS)
    assert_close(b, a, 0.02)                                            # the same numbers in other slots: only the order of sums differs


def test_fp8_cache_stays_near_bf16():
    """e4m3 keys and values are off by up to 2^-4 each; averaged over head_dim and positions far less reaches the logits."""
    assert_close(logits_after(engine(kv="fp8"), TOKENS), logits_after(engine(chunk=8), TOKENS), 0.25)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_a_short_window_forgets(kv):
    """One layer, window 8, no sinks: after 8 other tokens the first ones leave no trace in the logits."""
    a = engine(layers=1, kv=kv, window=8)
    x = logits_after(a, TOKENS[:20] + TOKENS[30:38])[-1]
    y = logits_after(a, TOKENS[5:7] + TOKENS[20:23] + TOKENS[5:20] + TOKENS[30:38])[-1]      # other tokens in front, the same positions
    assert torch.equal(x, y)
    z = engine(layers=1, kv=kv, window=8, sinks=2)
    x = logits_after(z, TOKENS[:20] + TOKENS[30:38])[-1]
    y = logits_after(z, TOKENS[:2] + TOKENS[20:23] + TOKENS[5:20] + TOKENS[30:38])[-1]       # the same first two, others behind them
    assert torch.equal(x, y)
    y = logits_after(z, TOKENS[3:5] + TOKENS[20:23] + TOKENS[5:20] + TOKENS[30:38])[-1]
    assert not torch.equal(x, y)


def test_a_session_longer_than_its_cache_in_a_graph():
    eng = engine(max_len=512, kv="fp8", window=32, sinks=4)
    assert eng.cache.capacity == 36
    eng.prefill(TOKENS); eager = eng.generate(100).tolist()
    eng.capture()
    eng.prefill(TOKENS); replay = eng.generate(100).tolist()
    assert eager == replay and int(eng.pos.item()) == 140


@pytest.mark.parametrize("layout", [0, 2])
@pytest.mark.parametrize("kw", [dict(chunk=8), dict(kv="fp8"), dict(kv="fp8", window=16, sinks=2, chunk=8)], ids=lambda k: "-".join(k))
def test_dependent_launches_change_nothing(kw, layout):
    """Kernels that start before the ones in front of them have ended, eager and captured: the same bits."""
    a, b = engine(layout, **kw), engine(layout, dependent_launch=True, **kw)
    assert torch.equal(logits_after(a, TOKENS), logits_after(b, TOKENS))
    a.prefill(TOKENS); b.prefill(TOKENS); b.capture()
    assert a.generate(30).tolist() == b.generate(30).tolist() and torch.equal(a.logits, b.logits)


@pytest.mark.parametrize("kv,window,sinks", [("bf16", 0, 0), ("fp8", 0, 0), ("fp8", 24, 3)])
@pytest.mark.parametrize("layout", [0, 2])
def test_chunks_agree_with_single_tokens(kv, window, sinks, layout):
    one, many = engine(layout, kv=kv, window=window, sinks=sinks, chunk=16), engine(layout, kv=kv, window=window, sinks=sinks, chunk=16)
    want = logits_after(one, TOKENS)
    many.reset()
    best = many.extend(TOKENS)                                          # 16 + 16 + 8
    many._check_status()
    got = many.logits_rows.float()
    assert_close(got, want[32:], 0.15)
    assert torch.equal(best[32:], got.argmax(-1)) and int(many.cur) == int(best[-1]) and int(many.pos) == 40
    many.cur.fill_(7); one.cur.fill_(7)
    many.forward_token(); one.forward_token()
    assert_close(many.logits.float(), one.logits.float(), 0.15)         # and the cache they leave behind serves the next token


def margin(row):
    top = row.topk(2).values
    return (top[0] - top[1]).item()


@pytest.mark.parametrize("kv,window,sinks", [("bf16", 0, 0), ("fp8", 40, 4)])
def test_verified_drafts_continue_as_greedy_decoding_would(kv, window, sinks):
    """Drafts made from the engine's own continuation, with wrong branches between them: the accepted path is the continuation,
    up to a near-tie (the chunk's and the single token's sums have another order), and decoding goes on from there."""
    eng = engine(kv=kv, window=window, sinks=sinks, chunk=16, max_len=256)
    eng.prefill(TOKENS[:20], chunked=True)
    first = int(eng.cur)
    truth = eng.generate(9).tolist()
    eng.prefill(TOKENS[:20], chunked=True)
    assert int(eng.cur) == first
    wrong = lambda t: (t + 1) % 2048
    drafts = [wrong(truth[0]), truth[0], wrong(truth[1]), truth[1], truth[2], wrong(truth[3])]
    parents = [-1, -1, 1, 1, 3, 4]
    new = eng.verify(drafts, parents)
    rows = eng.logits_rows.float()
    near = [margin(rows[i]) <= 2.0 ** -5 * rows[i].abs().max().item() for i in (0, 2, 4, 5)]
    n = len(new)
    assert 1 <= n <= 4 and int(eng.pos) == 20 + n and eng.log[:n].tolist() == new and int(eng.cur) == new[-1]
    for i in range(4):                                                  # token by token, as far as nothing was near a tie
        if near[i]: return
        assert new[i] == truth[i]
    after = eng.generate(5).tolist()
    one = logits_after(engine(kv=kv, window=window, sinks=sinks, chunk=16, max_len=256), TOKENS[:20] + [first] + truth[:4] + after[:4])[-5:]
    for row, got in zip(one, after):
        if margin(row) <= 2.0 ** -5 * row.abs().max().item(): return
        assert int(row.argmax()) == got


@pytest.mark.parametrize("kv,sinks", [("bf16", 0), ("bf16", 3), ("fp8", 0)])
def test_a_path_longer_than_the_window_is_verified_as_single_tokens_would(kv, sinks):
    """One layer, a window of 4, twelve right drafts in a chain: the logits behind each of them are those of the token decoded
    alone.  Ten roundings to bf16 in both (2^-8 / sqrt(3) each, independent) are 0.7 % of the logits' root mean square, and with the
    codes that a rounding flips to their neighbour (one of 32, by 2^-3) 1.2 %; the largest of 13 x 2048 such errors is 4.5 of them,
    the largest logit some 3.5 root mean squares: 0.016, and 0.04 leaves room."""
    eng = engine(layers=1, kv=kv, window=4, sinks=sinks, chunk=16, max_len=64)
    eng.prefill(TOKENS[:20], chunked=True)
    first = int(eng.cur)
    truth = eng.generate(12).tolist()
    eng.prefill(TOKENS[:20], chunked=True)
    new = eng.verify(truth, list(range(-1, 11)))
    rows = eng.logits_rows.float()
    want = logits_after(engine(layers=1, kv=kv, window=4, sinks=sinks, chunk=16, max_len=64), TOKENS[:20] + [first] + truth)[-13:]
    assert_close(rows, want, 0.04)
    for got, right, row in zip(new, truth, rows):
        if margin(row) <= 2.0 ** -5 * row.abs().max().item(): return
        assert got == right
    assert len(new) == 13 and int(eng.pos) == 33


@pytest.mark.parametrize("kw", [dict(), dict(chunk=8), dict(kv="fp8", chunk=8), dict(kv="fp8", window=16, sinks=2, chunk=8)], ids=lambda k: "-".join(k) or "plain")
def test_capture_leaves_a_live_session_as_it_was(kw):
    """Captured between two tokens of a session: what it holds, what it has logged and how it goes on are those of one that was not."""
    eager, eng = engine(**kw), engine(**kw)
    for e in (eager, eng): e.prefill(TOKENS[:12], chunked=bool(kw)); e.generate(3)
    held = lambda e: [e.cur, e.pos, e.step_no, e.log] + ([e.k_cache, e.v_cache] if e.cache is None else [t.view(torch.uint8) for t in (e.cache.k, e.cache.v, e.cache.k_exp, e.cache.v_exp) if t is not None])
    eng.capture()
    for a, b in zip(held(eng), held(eager)): assert torch.equal(a, b)
    assert eng.generate(6).tolist() == eager.generate(6).tolist()
    for a, b in zip(held(eng) + [eng.logits], held(eager) + [eager.logits]): assert torch.equal(a, b)


def test_a_token_drafted_twice_is_followed_where_it_leads_on():
    eng = engine(chunk=8)
    eng.prefill(TOKENS[:10], chunked=True)
    truth = eng.generate(3).tolist()
    eng.prefill(TOKENS[:10], chunked=True)
    new = eng.verify([truth[0], (truth[1] + 1) % 2048, truth[0], truth[1]], [-1, 0, -1, 2])
    for got, right, row in zip(new, truth, eng.logits_rows.float()[[0, 3, 4]]):
        if margin(row) <= 2.0 ** -5 * row.abs().max().item(): return
        assert got == right
    assert len(new) == 3 and int(eng.pos) == 13


def test_drafts_that_are_all_wrong_leave_the_next_token():
    eng = engine(chunk=8)
    eng.prefill(TOKENS[:10], chunked=True)
    pos = int(eng.pos)
    truth = int(eng.generate(1)[0])
    eng.prefill(TOKENS[:10], chunked=True)
    new = eng.verify([(truth + 1) % 2048, (truth + 2) % 2048], [-1, 0])
    if margin(eng.logits_rows[0].float()) > 2.0 ** -5 * eng.logits_rows[0].float().abs().max().item(): assert new == [truth]
    assert len(new) == 1 and int(eng.pos) == pos + 1
    assert len(eng.verify([], [])) == 1


def test_what_the_engine_refuses():
    plain, eng = engine(), engine(chunk=4, max_len=16)
    with pytest.raises(ValueError, match="chunk > 0"): plain.extend([1, 2])
    with pytest.raises(ValueError, match="parent"): eng.verify([1, 2], [-1])
    with pytest.raises(ValueError, match="comes before"): eng.verify([1, 2], [-1, 5])
    with pytest.raises(ValueError, match="at once"): eng.verify([1, 2, 3, 4], [-1, 0, 1, 2])
    with pytest.raises(ValueError, match="do not fit"): eng.extend(list(range(17)))
    with pytest.raises(ValueError, match="no tokens"): eng.extend([])
    with pytest.raises(ValueError, match="sinks"): engine(sinks=3)
    with pytest.raises(ValueError, match="elem"): engine(kv="int8")


def test_token_ids_outside_the_vocabulary_are_refused():
    """Their embedding rows would be whatever lay in the buffer."""
    eng = engine(chunk=4, max_len=16)
    for ids in ([1, 2048], [-1], [5, -2048, 3]):
        with pytest.raises(ValueError, match="below 2048"): eng.extend(ids)
        with pytest.raises(ValueError, match="below 2048"): eng.verify(ids, [-1] * len(ids))
    assert int(eng.pos) == 0 and eng.extend([0, 2047]).numel() == 2


def test_a_reset_engine_has_forgotten_a_session_that_left_its_cache():
    eng = engine(kv="fp8", max_len=8, chunk=4)
    eng.prefill(TOKENS[:8], chunked=True)
    eng.forward_token()                                                 # position 8 of a cache of 8: refused by the kernels, reported by check()
    torch.cuda.synchronize()
    assert int(eng.cache.status) != 0
    want = engine(kv="fp8", max_len=8, chunk=4).prefill(TOKENS[:5], chunked=True)
    assert int(eng.prefill(TOKENS[:5], chunked=True)) == int(want)


def test_the_engine_reports_a_wait_that_ran_out_once():
    from nwc_b200 import _lib as L
    eng = engine(chunk=4, max_len=16)
    assert L.lib.nwc_kv_wait_probe(L.stream(), L.ptr(eng.cache.status)) == 0
    with pytest.raises(RuntimeError, match="gave up"): eng._check_status()
    eng._check_status()
    assert L.lib.nwc_kv_wait_probe(L.stream(), L.ptr(torch.zeros(1, dtype=torch.int32, device="cuda"))) == 0       # in the library's word alone
    with pytest.raises(RuntimeError, match="gave up"): eng._check_status()
    eng._check_status()


@pytest.mark.parametrize("call", [lambda e: e.extend(TOKENS[:6]), lambda e: e.prefill(TOKENS[:6], chunked=True), lambda e: e.verify(TOKENS[:2], [-1, 0])], ids=["extend", "prefill", "verify"])
def test_keys_that_are_not_finite_are_reported_by_the_call_that_made_them(call):
    eng = engine(chunk=4, max_len=32)
    eng.w.layers[1]["k_norm"][3] = float("nan")
    with pytest.raises(RuntimeError, match="finite"): call(eng)
    eng.w.layers[1]["k_norm"][3] = 1.0
    eng.reset()
    assert int(eng.prefill(TOKENS[:6], chunked=True)) == int(eng.cur) and int(eng.pos) == 6


@pytest.mark.parametrize("H,rows", [(256, 1), (1000, 3), (8192, 70)])
def test_row_kernels_equal_the_single_row_ones(H, rows):
    from nwc_b200 import _lib as L
    g = torch.Generator().manual_seed(H)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    h, d, w, gu = bf(rows, H), bf(rows, H), bf(H), bf(rows, 2 * H)
    h2, xn, act = h.clone(), torch.empty_like(h), torch.empty_like(h)
    assert L.lib.nwc_add_rmsnorm_rows(L.stream(), L.ptr(h2), L.ptr(d), L.ptr(h2), L.ptr(w), 1e-6, H, rows, L.ptr(xn)) == 0
    assert L.lib.nwc_swiglu_rows(L.stream(), L.ptr(gu), H, rows, L.ptr(act)) == 0
    best = torch.empty(rows, dtype=torch.int64, device="cuda")
    tied = gu.clone(); tied[:, H // 2] = tied[:, 3] = tied.max() + 1
    assert L.lib.nwc_argmax_rows(L.stream(), L.ptr(tied), 2 * H, rows, L.ptr(best)) == 0
    assert (best == 3).all()
    for r in range(rows):
        a, x, s = h[r].clone(), torch.empty_like(w), torch.empty_like(w)
        assert L.lib.nwc_add_rmsnorm(L.stream(), L.ptr(a), L.ptr(d[r]), L.ptr(a), L.ptr(w), 1e-6, H, L.ptr(x), None) == 0
        assert L.lib.nwc_swiglu(L.stream(), L.ptr(gu[r]), H, L.ptr(s), None) == 0
        assert torch.equal(a, h2[r]) and torch.equal(x, xn[r]) and torch.equal(s, act[r])
