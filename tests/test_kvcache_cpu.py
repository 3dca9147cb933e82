"""Key/value cache: what its entry points refuse before anything touches the GPU, the masks of a draft tree, and the 64-bit
restatement that the GPU tests rely on, checked against elementary cases."""
import ctypes

import pytest
import torch

import kv_reference as R

A = 1 << 20                                                            # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from nwc_b200 import _lib
    return _lib


def cache(L, **kw):
    f = dict(k=A, v=A, k_exp=None, v_exp=None, layers=2, n_kv=2, head_dim=128, capacity=64, window=0, sinks=0, elem=0)
    f.update(kw)
    return ctypes.byref(L.KvCache(*[f[n] for n, _ in L.KvCache._fields_]))


BAD_CACHES = [dict(head_dim=96), dict(head_dim=0), dict(n_kv=0), dict(layers=0), dict(capacity=0), dict(elem=2), dict(k=None), dict(v=A + 8), dict(elem=1),
              dict(elem=1, k_exp=A), dict(window=64, sinks=1), dict(window=64), dict(window=10, sinks=64), dict(capacity=0x7FFFFF01), dict(capacity=2)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_caches_that_no_kernel_addresses(L, bad):
    """(capacity 2 and a window of 64 of 64 slots: right for one token, refused for the three of the call)"""
    c = cache(L, **bad)
    assert L.lib.nwc_kv_append(None, c, 0, A, 1024, 3, 4, None, None, A, A, 99, A, None, 1e-6, A, A) == -1
    assert L.lib.nwc_kv_attention(None, c, 0, A, 512, 3, 4, A, None, None, 0.1, A, None, 0, A) == -1
    if "capacity" not in bad or bad["capacity"] != 2:
        assert L.lib.nwc_kv_commit(None, c, 3, A, A, A, 2, A) == -1


def test_append_refusals(L):
    good = dict(layer=0, qkv=A, ld=1024, T=3, n_q=4, qn=None, kn=None, cos=A, sin=A, rows=99, pos=A, depth=None, eps=1e-6, out=A, status=A)
    for bad in (dict(layer=2), dict(qkv=None), dict(qkv=A + 2), dict(ld=1016), dict(ld=1028), dict(T=0), dict(T=65536), dict(n_q=0), dict(n_q=3), dict(qn=A), dict(kn=A),
                dict(cos=None), dict(sin=None), dict(cos=A + 8), dict(pos=None), dict(out=None), dict(out=A + 4), dict(status=None), dict(T=65)):
        a = {**good, **bad}
        assert L.lib.nwc_kv_append(None, cache(L), *a.values()) == -1, bad


def test_attention_refusals(L):
    good = dict(layer=0, q=A, ld=512, T=3, n_q=4, pos=A, visible=None, depth=None, scale=0.1, out=A, work=None, size=0, status=A)
    for bad in (dict(layer=2), dict(work=A + 8), dict(q=None), dict(q=A + 8), dict(ld=504), dict(ld=516), dict(T=0), dict(T=65), dict(n_q=0), dict(n_q=5), dict(pos=None), dict(visible=A), dict(depth=A),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None), dict(out=A + 2), dict(status=None)):
        a = {**good, **bad}
        assert L.lib.nwc_kv_attention(None, cache(L), *a.values()) == -1, bad
    a = {**good, "T": 1025, "visible": A, "depth": A}
    assert L.lib.nwc_kv_attention(None, cache(L, capacity=4096), *a.values()) == -1


def test_read_and_commit_refusals(L):
    for first, count in ((0, 0), (0, 65), (64, 1), (0xFFFFFFFF, 2)):
        assert L.lib.nwc_kv_read(None, cache(L), 0, first, count, A, A) == -1
    ring = cache(L, window=20, sinks=4)
    for first, count in ((4, 61), (100, 61), (0, 65), (0x7FFFFFFF, 1)):
        assert L.lib.nwc_kv_read(None, ring, 0, first, count, A, A) == -1
    assert L.lib.nwc_kv_read(None, cache(L), 0, 0, 4, A + 8, A) == -1 and L.lib.nwc_kv_read(None, cache(L), 0, 0, 4, A, None) == -1
    for T, most, path in ((0, 0, A), (1025, 3, A), (3, 4, A), (3, 3, None), (65, 3, A)):
        assert L.lib.nwc_kv_commit(None, cache(L), T, A, path, A, most, A) == -1
    assert L.lib.nwc_kv_commit(None, cache(L), 3, A, A, A, 0, A) == 0                       # an empty path: nothing to launch


def test_python_refusals():
    from nwc_b200 import KVCache
    bf = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    codes, byte = torch.zeros(1, 2, 8, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(1, 2, 8, dtype=torch.uint8)
    for args, kw, text in (((bf, bf[:, :1]), {}, "one type"), ((bf.float(), bf.float()), {}, "bfloat16 or float8"), ((bf.transpose(1, 2), bf.transpose(1, 2)), {}, "contiguous"),
                           ((codes, codes), {}, "exponent bytes"), ((bf, bf, byte, byte), {}, "exponent bytes"), ((codes, codes, byte, byte[:, :, :4]), {}, "exponent bytes are"),
                           ((bf[..., :32].contiguous(), bf[..., :32].contiguous()), {}, "head_dim"), ((bf, bf), dict(window=-1), "negative"), ((bf, bf), dict(sinks=2), "need a window"),
                           ((bf, bf), dict(window=8, sinks=1), "capacity of 9"), ((bf, bf), {}, "CUDA")):
        with pytest.raises(ValueError, match=text): KVCache.over(*args, **kw)


def test_draft_tree_masks():
    from nwc_b200 import draft_tree
    parents = [-1, 0, 0, 2, -1] + [4 + i for i in range(40)]
    visible, depth = draft_tree(parents, "cpu")
    assert visible.shape == (45, 2) and depth.tolist()[:6] == [0, 1, 1, 2, 0, 1] and int(depth[-1]) == 40
    for t in range(45):
        seen, at = set(), t
        while at >= 0: seen.add(at); at = parents[at]
        assert {j for j in range(45) if (int(visible[t, j // 32]) >> (j % 32)) & 1} == seen
    for bad in ([], [0], [-1, 1], [-1, -2], list(range(-1, 1024))):
        with pytest.raises(ValueError): draft_tree(bad, "cpu")


def test_reference_rounding_is_that_of_the_type():
    y = torch.cat([torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double(), torch.linspace(-448, 448, 20001, dtype=torch.float64),
                   torch.linspace(-0.03, 0.03, 20001, dtype=torch.float64)])
    y = y[torch.isfinite(y)].float().double()
    assert torch.equal(R.rounded_e4m3(y), y.float().to(torch.float8_e4m3fn).double())
    x = torch.tensor([[448.0], [449.0], [0.0], [447.0], [224.0], [225.0], [1e-45]])
    assert R.unit_exponent(x).tolist() == [0, 1, -127, 0, -1, 0, -127]


def test_reference_attention_in_a_case_done_by_hand():
    k = torch.tensor([[[0.0], [0.0], [9.0], [0.0]]], dtype=torch.float64); v = torch.tensor([[[1.0], [3.0], [100.0], [8.0]]], dtype=torch.float64)
    q = torch.tensor([[[1.0]], [[1.0]]], dtype=torch.float64)
    out, weight = R.attend(q, k, v, pos=0)
    assert out.flatten().tolist() == [1.0, 2.0] and weight.flatten().tolist() == [1.0, 2.0]
    out, _ = R.attend(q, k, v, pos=0, visible=R.tree_bits(2, [[], [1]]), depth=torch.tensor([0, 0]))
    assert out.flatten().tolist() == [0.0, 3.0]
    # ring of three behind one sink: position 4 lives in slot 1, 5 in slot 2
    out, _ = R.attend(q[:1], k, v, pos=4, window=1, sinks=1)
    assert out.item() == 2.0


def test_the_wait_probe_refuses_no_status_word(L):
    assert L.lib.nwc_kv_wait_probe(None, None) == -1


@pytest.mark.parametrize("window,sinks,pos", [(8, 0, None), (1, 0, 0), (3, 2, 0), (3, 4, 1), (8, 5, 90), (64, 0, None)])
def test_draft_tree_masks_under_a_window(window, sinks, pos):
    """A draft sees the ancestors that the same token sees when it stands alone behind its path."""
    from nwc_b200 import draft_tree
    parents = [-1, 0, 0, 2, -1] + [4 + i for i in range(40)] + [20, 45, 7]
    visible, depth = draft_tree(parents, "cpu", window=window, sinks=sinks, pos=pos)
    for t in range(len(parents)):
        seen, at = set(), t
        while at >= 0:
            if depth[t] - depth[at] < window or (sinks and pos + depth[at] < sinks): seen.add(at)
            at = parents[at]
        assert {j for j in range(len(parents)) if (int(visible[t, j // 32]) >> (j % 32)) & 1} == seen
    for bad in (dict(window=-1), dict(sinks=2), dict(window=4, sinks=-1), dict(window=4, sinks=1)):
        with pytest.raises(ValueError): draft_tree([-1, 0], "cpu", **bad)


@pytest.mark.parametrize("window,sinks,pos", [(8, 0, 30), (8, 3, 30), (4, 3, 1), (1, 0, 0)])
def test_a_chain_longer_than_the_window_sees_what_single_tokens_see(window, sinks, pos):
    from nwc_b200 import draft_tree
    T, n_q, n_kv, hd = 12, 2, 1, 64
    g = torch.Generator().manual_seed(window + pos)
    k, v = torch.randn(2, n_kv, sinks + window + T, hd, generator=g, dtype=torch.float64)
    q = torch.randn(T, n_q, hd, generator=g, dtype=torch.float64)
    visible, depth = draft_tree([t - 1 for t in range(T)], "cpu", window=window, sinks=sinks, pos=pos)
    tree, _ = R.attend(q, k, v, pos, window, sinks, visible, depth)
    chunk, _ = R.attend(q, k, v, pos, window, sinks)
    assert (tree - chunk).abs().max() < 1e-12


def test_the_longest_accepted_path_of_a_draft_tree():
    from nwc_b200.decode import accepted_path as path
    assert path([], [], [7]) == [0] and path([5, 6], [-1, 0], [7, 1, 1]) == [0]
    assert path([7, 8, 9], [-1, 0, 1], [7, 8, 1, 1]) == [0, 1, 2]                            # the third draft is wrong
    assert path([7, 7, 8], [-1, -1, 1], [7, 8, 8, 4]) == [0, 2, 3]                           # drafted twice, the second leads on
    assert path([7, 8, 7, 8], [-1, 0, -1, 2], [7, 8, 4, 8, 4]) == [0, 1, 2]                  # both do: the first
    assert path([7, 3, 9, 9], [-1, 0, 1, 0], [7, 4, 9, 1, 1]) == [0, 1]                      # a child of a wrong draft counts for nothing


def fake_cache(L, **kw):
    """A KVCache whose tensors nobody looks at: what its calls refuse before they reach the device."""
    from nwc_b200 import KVCache
    c = KVCache.__new__(KVCache)
    f = dict(layers=1, n_kv=2, capacity=64, head_dim=128, window=20, sinks=4, elem="bf16", _at=0, device=torch.device("cuda:0"), status=None, _status=A, _need={})
    f.update(kw)
    for name, value in f.items(): setattr(c, name, value)
    c._ref = cache(L, window=c.window, sinks=c.sinks)
    return c


def test_numbers_that_do_not_fit_the_calls_are_refused_not_cut(L):
    """2^32 + 5 would arrive as 5."""
    ring = fake_cache(L)
    for first, count in ((2 ** 32 + 5, 1), (2 ** 31 - 1, 1), (5, 2 ** 32), (2 ** 63, 2)):
        with pytest.raises(ValueError, match="positions"): ring.read(first, count)

    class Int32:                                                        # a path, a count and a position on the device
        dtype = torch.int32
        def __init__(self, n): self.n = n
        def dim(self): return 1
        def numel(self): return self.n
        def get_device(self): return 0
        def is_contiguous(self): return True
        def data_ptr(self): return A
    for tokens in (0, -1, 1025, 2 ** 32 + 4):
        with pytest.raises(ValueError, match="1 to 1024"): ring.commit(Int32(1), Int32(3), Int32(1), tokens=tokens)


def test_scales_that_leave_the_numbers_are_refused(L):
    """The kernels work with scale x log2(e): 2.9e38 would become infinite."""
    for scale in (2.9e38, 2.4e38, 0.0, -0.5):
        assert L.lib.nwc_kv_attention(None, cache(L), 0, A, 512, 3, 4, A, None, None, scale, A, None, 0, A) == -1


def test_the_stride_of_a_single_row_does_not_matter(L):
    c = fake_cache(L, _at=-1)
    row = torch.zeros(1024, dtype=torch.bfloat16)
    for stride in (1024, 1, 0, 12):
        assert c._tokens(row.as_strided((1, 1024), (stride, 1)), 2, "qkv") == (1, 1024)
    with pytest.raises(ValueError): c._tokens(row.as_strided((2, 64), (12, 1)), 2, "qkv")


def test_tensors_that_want_gradients_are_refused_while_gradients_are_on(L):
    c = fake_cache(L, _at=-1)
    x = torch.zeros(2, 1024, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="no_grad"): c._tokens(x, 2, "qkv")
    with torch.no_grad(): assert c._tokens(x, 2, "qkv") == (2, 1024)
    assert c._tokens(x.detach(), 2, "qkv") == (2, 1024)


@pytest.mark.parametrize("answer", [None, lambda shape, dtype: None, lambda shape, strides, dtype: torch.empty(shape, dtype=dtype), lambda shape, strides, dtype: torch.empty(shape)],
                         ids=["gone", "other arguments", "other device", "other type"])
def test_torchs_own_allocation_is_used_only_where_it_answers_as_the_public_one(monkeypatch, answer):
    from nwc_b200 import kvcache
    guards = torch._C._dynamo.guards
    if answer is None: monkeypatch.delattr(guards, "_empty_strided_cuda", raising=False)
    else: monkeypatch.setattr(guards, "_empty_strided_cuda", answer, raising=False)
    kvcache._allocation.cache_clear()
    try: assert kvcache._allocation() is kvcache._plain_empty
    finally: kvcache._allocation.cache_clear()


def test_a_draft_tree_reads_its_parents_once():
    """They may lie on a device, where every number read is a wait."""
    from nwc_b200 import draft_tree
    class Parents(list):
        read = 0
        def __iter__(self):
            for p in list.__iter__(self): self.read += 1; yield p
        def __getitem__(self, i): self.read += 1; return list.__getitem__(self, i)
    parents = Parents(range(-1, 63))
    draft_tree(parents, "cpu", window=20)
    assert parents.read == 64


def test_row_kernel_refusals(L):
    for bad in (dict(h=None), dict(out=None), dict(w=None), dict(H=0), dict(rows=0), dict(xn=None)):
        a = {**dict(h=A, delta=None, out=A, w=A, eps=1e-6, H=256, rows=3, xn=A), **bad}
        assert L.lib.nwc_add_rmsnorm_rows(None, *a.values()) == -1, bad
    for bad in (dict(gu=None), dict(I=0), dict(rows=0), dict(rows=65536), dict(a=None)):
        assert L.lib.nwc_swiglu_rows(None, *{**dict(gu=A, I=256, rows=3, a=A), **bad}.values()) == -1, bad
    for bad in (dict(logits=None), dict(V=0), dict(rows=0), dict(best=None)):
        assert L.lib.nwc_argmax_rows(None, *{**dict(logits=A, V=256, rows=3, best=A), **bad}.values()) == -1, bad
