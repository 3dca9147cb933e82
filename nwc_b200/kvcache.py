"""Key/value cache for long sessions and for several tokens at once: bf16 or quantised as it is written (e4m3 codes with one
power-of-two scale per row), plain or a ring under a sliding window whose first tokens ("sinks") stay visible, read by one
token, by a chunk of a prompt or by a tree of drafted tokens.  One call = one or two kernels of this library on the current
stream; positions live in device memory, so every call can be captured in a CUDA graph.

    cache = KVCache(n_kv=8, head_dim=128, capacity=8192, elem="fp8", layers=36)
    q = cache.append(qkv, pos, cos, sin, q_norm, k_norm, layer=i)        # T tokens at positions pos .. pos + T - 1
    out = cache.attend(q, pos, layer=i)                                  # [T, n_q * head_dim]

A draft tree is verified with the same two calls and the masks of `draft_tree` (which takes the cache's window), then `commit`
moves the accepted path together.
"""
import ctypes
import functools
import math

import torch

from . import _lib as L

BF16, INT32 = torch.bfloat16, torch.int32
current_device, raw_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)     # (absent without CUDA)
MAX_TREE, MAX_POSITIONS = 1024, 0x7FFFFFFF
ELEMS = {"bf16": (0, torch.bfloat16), "fp8": (1, torch.float8_e4m3fn)}
STATUS_TEXT = ((1, "a position outside the cache or the rotary tables"), (2, "a key or value that is not finite"), (4, "an accepted path that is not one"),
               (8, "a bounded wait inside the attention gave up, its outputs are not valid"))


def _plain_empty(shape, strides, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


@functools.cache
def _allocation():
    """An allocation on the current device that does not go through the dispatcher (0.8 us instead of 1.9).  It is no public name
    of torch: taken once it has answered as torch.empty does."""
    try:
        from torch._C._dynamo.guards import _empty_strided_cuda as direct
        t = direct((2, 3), (3, 1), BF16)
        if t.shape == (2, 3) and t.stride() == (3, 1) and t.dtype is BF16 and t.is_cuda and t.get_device() == torch.cuda.current_device(): return direct
    except Exception: pass
    return _plain_empty


def draft_tree(parents, device="cuda", window=0, sinks=0, pos=None):
    """Masks of a draft tree: parents[i] < i is the draft that token i continues, -1 where it continues the cached text.
    Returns (visible int32 [T, ceil(T / 32)], depth int32 [T]): every token sees its ancestors and itself.
    window, sinks: of the cache that the tree enters, at position pos (a number; needed beside sinks).  A token then sees the
    ancestors that it would see as a single token: the last `window` positions of its path and those below `sinks`."""
    T = len(parents)
    if not T: raise ValueError("a draft tree has at least one token")
    if T > MAX_TREE: raise ValueError(f"a draft tree has at most {MAX_TREE} tokens, not {T}")
    if window < 0 or sinks < 0 or sinks and not window: raise ValueError("window and sinks are not negative, and sinks need a window")
    if sinks and pos is None: raise ValueError("beside sinks, pos says which drafts are among them")
    parents, masks, depth = [int(p) for p in parents], [], []
    for i, p in enumerate(parents):
        if not -1 <= p < i: raise ValueError(f"draft {i} hangs below draft {p}: a parent comes before its children (-1 = none)")
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
        if window and depth[i] >= window:                             # the ancestor that its parent saw last
            left = i
            for _ in range(window): left = parents[left]
            if not (sinks and pos + depth[left] < sinks): masks[i] &= ~(1 << left)
    words = [[(m >> 32 * w) & 0xFFFFFFFF for w in range((T + 31) // 32)] for m in masks]
    signed = [[w - (1 << 32) if w >> 31 else w for w in row] for row in words]
    return torch.tensor(signed, dtype=torch.int32, device=device), torch.tensor(depth, dtype=torch.int32, device=device)


class KVCache:
    """`layers` x `n_kv` heads x `capacity` slots of head_dim (64, 128 or 256) numbers for K and for V.

    window = 0: position p lives in slot p, a token sees every position up to its own.
    window > 0: a token sees the last `window` positions (its own among them) and the first `sinks`; slots beyond the sinks are
    taken in turn, so positions run on without end.  T tokens at once need capacity - sinks >= window + T - 1.

    The calls have no backward pass: with gradients enabled they refuse tensors that require them.

    Position tensors are int32 [1] on the cache's device.  Values that are not finite are stored as 0 and reported by check(),
    as are positions outside the cache."""

    def __init__(self, n_kv, head_dim, capacity, elem="bf16", layers=1, window=0, sinks=0, device="cuda"):
        L.require_cuda()
        _, dtype = _elem(elem)
        if min(layers, n_kv, head_dim, capacity) < 1: raise ValueError("layers, n_kv, head_dim and capacity are at least 1")
        shape = (layers, n_kv, capacity, head_dim)
        # zeros, not empty: a slot that no token has reached holds numbers
        zeros = lambda: torch.zeros(shape, dtype=torch.uint8 if elem == "fp8" else dtype, device=device).view(dtype)
        exps = (lambda: torch.zeros(shape[:3], dtype=torch.uint8, device=device)) if elem == "fp8" else (lambda: None)
        self._bind(zeros(), zeros(), exps(), exps(), window, sinks)

    @classmethod
    def over(cls, k, v, k_exp=None, v_exp=None, window=0, sinks=0):
        """A cache over tensors that the caller holds: k, v [layers, n_kv, capacity, head_dim] bf16, or float8_e4m3fn with the
        rows' exponent bytes k_exp, v_exp uint8 [layers, n_kv, capacity]."""
        self = cls.__new__(cls)
        self._bind(k, v, k_exp, v_exp, window, sinks)
        return self

    def _bind(self, k, v, k_exp, v_exp, window, sinks):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device: raise ValueError("k and v are [layers, n_kv, capacity, head_dim] of one type on one device")
        if k.dtype not in (torch.bfloat16, torch.float8_e4m3fn): raise ValueError(f"a cache holds bfloat16 or float8_e4m3fn, not {k.dtype}")
        quantised = k.dtype == torch.float8_e4m3fn
        if not (k.is_contiguous() and v.is_contiguous()): raise ValueError("k and v are contiguous")
        for t in (k_exp, v_exp):
            if quantised != (t is not None): raise ValueError("fp8 caches come with exponent bytes, bf16 caches without")
            if quantised and (t.dtype != torch.uint8 or t.shape != k.shape[:3] or not t.is_contiguous() or t.device != k.device): raise ValueError("exponent bytes are contiguous uint8 [layers, n_kv, capacity] beside the codes")
        self.layers, self.n_kv, self.capacity, self.head_dim = k.shape
        if self.head_dim not in (64, 128, 256): raise ValueError(f"head_dim is 64, 128 or 256, not {self.head_dim}")
        window, sinks = int(window), int(sinks)
        if window < 0 or sinks < 0: raise ValueError("window and sinks are not negative")
        if not window and sinks: raise ValueError("sinks need a window")
        if window and self.capacity - sinks < window: raise ValueError(f"a window of {window} behind {sinks} sinks needs a capacity of {window + sinks} at least, not {self.capacity}")
        if self.capacity > 0x7FFFFF00: raise ValueError("capacity is below 2^31 - 256")
        if not k.is_cuda: raise ValueError("a cache lives on a CUDA device")
        if k.data_ptr() % 16 or v.data_ptr() % 16: raise ValueError("k and v are 16-byte aligned")
        self.window, self.sinks, self.elem = window, sinks, "fp8" if quantised else "bf16"
        self.k, self.v, self.k_exp, self.v_exp, self.device = k, v, k_exp, v_exp, k.device
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        at = lambda t: None if t is None else t.data_ptr()
        self._c = L.KvCache(at(k), at(v), at(k_exp), at(v_exp), self.layers, self.n_kv, self.head_dim, self.capacity, window, sinks, 1 if quantised else 0)
        self._at = k.get_device()
        with torch.cuda.device(self._at): L.lib.nwc_setup(); self._strided = _allocation()           # not in the first call, which may be one that is captured
        self._need = {}                                               # workspace bytes per (tokens, query heads)
        self._ref, self._status = ctypes.byref(self._c), self.status.data_ptr()

    # ---- calls ----
    def append(self, qkv, pos, cos, sin, q_norm=None, k_norm=None, eps=1e-6, depth=None, layer=0):
        """Store T tokens of a fused projection qkv [T, (n_q + 2 n_kv) head_dim] (bf16; a vector is one token) at positions
        pos .. pos + T - 1: per-head RMSNorm of q and k (with both weights), rotary embedding with rows of the bf16 tables cos /
        sin [positions, head_dim] - row pos + depth[t] for drafts, pos + t otherwise - and one rounding to the cache's type.
        Returns the queries, bf16 [T, n_q, head_dim]."""
        if qkv.dim() == 1: qkv = qkv[None]
        T, width = self._tokens(qkv, 2, "qkv")
        hd, at, n_kv = self.head_dim, self._at, self.n_kv
        n_q = width // hd - 2 * n_kv
        if width % hd or n_q <= 0 or n_q % n_kv: raise ValueError(f"qkv rows of {width} are not (n_q + 2 * {n_kv}) heads of {hd}, n_q a multiple of {n_kv}")
        rows = cos.shape[0]
        if cos.shape != (rows, hd) or sin.shape != (rows, hd): raise ValueError(f"cos and sin are both [positions, {hd}]")
        if cos.dtype is not BF16 or sin.dtype is not BF16 or cos.get_device() != at or sin.get_device() != at or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError(f"cos and sin are contiguous bf16 on {self.device}")
        qn = kn = dp = None
        if q_norm is not None and k_norm is not None:
            for t in (q_norm, k_norm):
                if t.requires_grad: self._no_grad("q_norm and k_norm")
                if t.dtype is not BF16 or t.get_device() != at or t.shape != (hd,) or not t.is_contiguous(): raise ValueError(f"q_norm and k_norm are contiguous bf16 [{hd}] on {self.device}")
            qn, kn = q_norm.data_ptr(), k_norm.data_ptr()
        elif q_norm is not None or k_norm is not None: raise ValueError("q_norm and k_norm come together")
        if depth is not None: self._int32(depth, T, "depth"); dp = depth.data_ptr()
        self._int32(pos, 1, "pos")
        if not 0 <= layer < self.layers: self._layer(layer)
        out = self._empty((T, n_q, hd), (n_q * hd, hd, 1))
        self._call("nwc_kv_append", L.lib.nwc_kv_append, self._ref, layer, qkv.data_ptr(), qkv.stride(0) if T > 1 else width, T, n_q, qn, kn, cos.data_ptr(), sin.data_ptr(), rows,
                   pos.data_ptr(), dp, eps, out.data_ptr(), self._status)
        return out

    def attend(self, q, pos, visible=None, depth=None, layer=0, scale=None):
        """Attention of T stored tokens at positions pos .. pos + T - 1 (q [T, n_q, head_dim], bf16) over what each of them
        sees; with the masks of draft_tree (made with this cache's window and sinks) the tokens are drafts (at most 1024).  Returns bf16 [T, n_q * head_dim]; a token that
        sees nothing gets zeros.  scale: of the scores, positive, 1 / sqrt(head_dim) by default."""
        T, n_q, hd = self._tokens(q, 3, "q")
        if hd != self.head_dim or n_q % self.n_kv or n_q > 1 and q.stride(1) != hd: raise ValueError(f"q is [T, n_q, {self.head_dim}] with n_q a multiple of {self.n_kv} and a token's heads side by side")
        if (visible is None) != (depth is None): raise ValueError("visible and depth come together (draft_tree makes them)")
        if visible is not None:
            if T > MAX_TREE: raise ValueError(f"a draft tree has at most {MAX_TREE} tokens, not {T}")
            self._int32(visible, T * ((T + 31) // 32), "visible"); self._int32(depth, T, "depth")
        self._int32(pos, 1, "pos")
        if not 0 <= layer < self.layers: self._layer(layer)
        if scale is None: scale = 1.0 / math.sqrt(hd)
        elif not 0.0 < scale <= 2e38: raise ValueError(f"scale is a positive number up to 2e38, not {scale}")
        out = self._empty((T, n_q * hd), (n_q * hd, 1))
        need = self._need.get((T, n_q))
        if need is None:
            with torch.cuda.device(self.device): need = self._need[T, n_q] = L.lib.nwc_kv_attention_workspace(self._ref, T, n_q)
        # a workspace of the call's own: the allocator keeps it from calls on other streams, a graph keeps it in its pool
        work = self._empty((need // 2,), (1,)) if need else None
        self._call("nwc_kv_attention", L.lib.nwc_kv_attention, self._ref, layer, q.data_ptr(), q.stride(0) if T > 1 else n_q * hd, T, n_q, pos.data_ptr(), None if visible is None else visible.data_ptr(),
                   None if depth is None else depth.data_ptr(), float(scale), out.data_ptr(), None if work is None else work.data_ptr(), need, self._status)
        return out

    def read(self, first, count, layer=0):
        """Positions first .. first + count - 1 of a layer as bf16 (K, V), each [n_kv, count, head_dim].  Of a ring, positions
        that it still holds."""
        first, count = int(first), int(count)
        if first < 0 or count < 1: raise ValueError("positions from 0 on, at least one")
        if not self.window and first + count > self.capacity: raise ValueError(f"positions {first} .. {first + count - 1} are outside a cache of {self.capacity}")
        if first + count > MAX_POSITIONS: raise ValueError(f"a session has at most {MAX_POSITIONS} positions")
        if self.window and first + count - max(first, self.sinks) > self.capacity - self.sinks: raise ValueError(f"{count} positions do not lie in a ring of {self.capacity - self.sinks} at the same time")
        if not 0 <= layer < self.layers: self._layer(layer)
        hd = self.head_dim
        shape, strides = (self.n_kv, count, hd), (count * hd, hd, 1)
        k, v = self._empty(shape, strides), self._empty(shape, strides)
        self._call("nwc_kv_read", L.lib.nwc_kv_read, self._ref, layer, first, count, k.data_ptr(), v.data_ptr())
        return k, v

    def commit(self, pos, path, count, tokens=None):
        """The accepted path of the draft tree stored at pos, in all layers: row path[i] of the drafts becomes row i for i <
        count (int32 [1]; path int32, strictly rising).  `tokens`: size of the tree (default: the largest that the
        cache could have taken), beyond which a path is refused.  The caller then advances pos by count."""
        if path.dim() != 1: raise ValueError("path is a vector of draft numbers")
        self._int32(path, path.numel(), "path"); self._int32(count, 1, "count"); self._int32(pos, 1, "pos")
        if tokens is None: tokens = min(MAX_TREE, self.capacity - self.sinks - self.window + 1 if self.window else self.capacity)
        if not 1 <= tokens <= MAX_TREE: raise ValueError(f"a draft tree has 1 to {MAX_TREE} tokens, not {tokens}")
        self._call("nwc_kv_commit", L.lib.nwc_kv_commit, self._ref, tokens, pos.data_ptr(), path.data_ptr(), count.data_ptr(), min(path.numel(), tokens), self._status)

    def check(self):
        """Waits for the device; raises when a call since the last check met one of STATUS_TEXT."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("key/value cache: " + "; ".join(text for bit, text in STATUS_TEXT if bits & bit))

    # ---- helpers (a call of one token takes microseconds on the device: what every call checks is kept to plain comparisons) ----
    def _tokens(self, t, dims, name):
        shape = t.shape
        if t.dim() != dims or t.dtype is not BF16 or t.get_device() != self._at or t.stride(-1) != 1 or t.stride(0) % 8 and shape[0] > 1 or t.data_ptr() % 16:
            raise ValueError(f"{name} is a {dims}-dimensional bf16 tensor on {self.device}, rows contiguous and 16-byte aligned")
        if t.requires_grad: self._no_grad(name)
        if not 0 < shape[0] <= 65535: raise ValueError(f"a call takes 1 to 65535 tokens, not {shape[0]}")
        return shape

    def _int32(self, t, n, name):
        if t.dtype is not INT32 or t.get_device() != self._at or t.numel() != n or not t.is_contiguous(): raise ValueError(f"{name} is int32 with {n} elements on {self.device}")

    def _empty(self, shape, strides):
        """bf16 on the cache's device."""
        return self._strided(shape, strides, BF16) if current_device() == self._at else torch.empty(shape, dtype=BF16, device=self.device)

    def _no_grad(self, name):
        if torch.is_grad_enabled(): raise ValueError(f"{name}: the cache's calls have no backward pass; call them under torch.no_grad()")

    def _layer(self, layer):
        raise IndexError(f"layer {layer} of a cache of {self.layers}")

    def _call(self, name, fn, *args):
        """One library call on the current stream of the cache's device."""
        if current_device() == self._at: err = fn(raw_stream(self._at), *args)
        else:
            with torch.cuda.device(self._at): err = fn(raw_stream(self._at), *args)
        if err == -1: raise ValueError(f"{name}: the cache ({self.capacity} slots, window {self.window}, {self.sinks} sinks) does not take this call")
        if err: raise RuntimeError(f"{name} error {err}")


def _elem(elem):
    if elem not in ELEMS: raise ValueError(f"elem is 'bf16' or 'fp8', not {elem!r}")
    return ELEMS[elem]
