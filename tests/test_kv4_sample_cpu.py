"""Argument checks of the 4-bit cache and sampling entries at the C-ABI boundary, on CPU (nothing is launched)."""
import ctypes

import pytest
import torch

from tokengate_b200 import _lib, ops
from tokengate_b200.kv4 import KV4Cache

BAD, NO, ALIGN = _lib.TG_ERR_INVALID_ARGUMENT, _lib.TG_ERR_UNSUPPORTED, _lib.TG_ERR_ALIGNMENT


def test_cache_bytes():
    L, n = _lib.lib(), ctypes.c_size_t(7)
    for cap, tiles in ((1, 1), (32, 1), (33, 2), (131072, 4096)):
        assert L.tg_kv4_cache_bytes(3, 8, cap, ctypes.byref(n)) == 0 and n.value == 3 * 8 * tiles * 4608
    assert L.tg_kv4_cache_bytes(3, 8, 0, ctypes.byref(n)) == BAD and n.value == 0
    assert L.tg_kv4_cache_bytes(3, 8, 5, None) == BAD


def _write(**over):
    a = dict(k=4096, k_sb=0, k_ss=256, k_sh=128, v=8192, v_sb=0, v_ss=256, v_sh=128, B=1, Hkv=2, D=128, start=0,
             count=5, cache=16384, capacity=8, stream=None)
    a.update(over)
    return list(a.values())


def test_write_and_read_checks():
    L = _lib.lib()
    for over, st in ((dict(cache=None), BAD), (dict(k=None), BAD), (dict(D=64), NO), (dict(B=0), BAD), (dict(Hkv=0), BAD),
                     (dict(start=-1), BAD), (dict(start=4), BAD), (dict(start=9, count=0), BAD), (dict(count=-1), BAD),
                     (dict(start=2 ** 62), BAD), (dict(capacity=2 ** 31), BAD), (dict(k=4098), ALIGN), (dict(v_ss=260), ALIGN),
                     (dict(cache=16392), ALIGN), (dict(count=0), 0)):
        assert L.tg_kv4_write(*_write(**over)) == st, over
    r = lambda *a: L.tg_kv4_read(*a)  # noqa: E731
    assert r(16384, 8, 1, 2, 128, 4, 5, 4096, 0, 256, 128, 8192, 0, 256, 128, None) == BAD
    assert r(16384, 8, 1, 2, 128, 0, 5, None, 0, 256, 128, 8192, 0, 256, 128, None) == BAD
    assert r(16384, 8, 1, 2, 128, 8, 0, None, 0, 0, 0, None, 0, 0, 0, None) == 0


def test_append_checks():
    def call(**over):
        a = dict(q=4096, ld_q=512, n_q=4, k=8192, ld_k=256, n_k=2, v=8192, ld_v=256, rows=1, qw=512, kw=512, cos=512,
                 sin=512, ld_cs=128, D=128, eps=1e-6, q_out=4096, ld_qo=512, cache=16384, cap=8, slot=64, stream=None)
        a.update(over)
        return _lib.lib().tg_qk_norm_rope_append_kv4(*a.values())
    for over, st in ((dict(q=None), BAD), (dict(slot=None), BAD), (dict(cache=None), BAD), (dict(D=96), NO), (dict(ld_q=500), BAD),
                     (dict(ld_v=128), BAD), (dict(n_q=0), BAD), (dict(rows=-1), BAD), (dict(q=4100), ALIGN), (dict(ld_k=258), ALIGN),
                     (dict(rows=0), 0)):
        assert call(**over) == st, over


def test_attention_checks():
    def call(**over):
        a = dict(q=4096, q_sb=0, q_sh=128, qs=None, qs_sb=0, cache=16384, cap=64, bias=None, b_sb=0, b_sh=0, n_valid=64,
                 n_prefix=5, n_keys=6, nk=None, out=4096, o_sb=0, o_sh=128, ws=None, wsb=0, B=1, Hq=4, Hkv=2, D=128,
                 scale=0.1, stream=None)
        a.update(over)
        return _lib.lib().tg_decode_attn_kv4(*a.values())
    for over, st in ((dict(q=None), BAD), (dict(out=None), BAD), (dict(n_valid=None), BAD), (dict(cache=None), BAD), (dict(n_prefix=7), BAD),
                     (dict(n_keys=0, n_prefix=0), BAD), (dict(n_keys=65), BAD), (dict(Hq=5), BAD), (dict(Hq=18), NO), (dict(D=64), NO),
                     (dict(scale=0.0), BAD), (dict(scale=float("nan")), BAD), (dict(cache=16392), ALIGN), (dict(B=70000), BAD)):
        assert call(**over) == st, over


def test_sample_checks():
    def call(**over):
        a = dict(logits=4096, dtype=1, stride=100, B=2, V=100, u=64, t=64, k=None, p=None, m=None, token=64, lp=None, stream=None)
        a.update(over)
        return _lib.lib().tg_sample(*a.values())
    for over, st in ((dict(logits=None), BAD), (dict(u=None), BAD), (dict(t=None), BAD), (dict(token=None), BAD), (dict(dtype=2), BAD),
                     (dict(V=0), BAD), (dict(stride=99), BAD), (dict(B=-1), BAD), (dict(B=70000), BAD), (dict(V=2 ** 19 + 1, stride=2 ** 20), NO),
                     (dict(logits=4097), ALIGN), (dict(dtype=0, logits=4098), ALIGN), (dict(B=0, logits=None), 0)):
        assert call(**over) == st, over


def test_packed_calls_are_the_calls():
    """tg_call with the arguments in one array: the same checks, its own for the entry and the count, and
    values outside an int's range refused instead of cut."""
    import struct
    L = _lib.lib()
    names = ["tg_kv4_write", "tg_kv4_read", "tg_qk_norm_rope_append_kv4", "tg_decode_attn_kv4", "tg_sample"]
    calls = [_lib.kv4_write, _lib.kv4_read, _lib.qk_norm_rope_append_kv4, _lib.decode_attn_kv4, _lib.sample]
    floats = [[], [], [15], [23], []]
    for e, (name, call) in enumerate(zip(names, calls)):
        sig = _lib._SIGNATURES[name]
        assert (call._entry, call._n) == (e, len(sig) - 1)
        assert [i for i, t in enumerate(sig) if t is ctypes.c_float] == floats[e]
        zeros = bytes(8 * call._n)
        n = call._n
        # empty sizes do nothing, all else of zeros is refused
        assert L.tg_call(e, zeros, n, None) == (0 if name in ("tg_sample", "tg_qk_norm_rope_append_kv4") else BAD)
        assert L.tg_call(e, zeros, n - 1, None) == BAD and b"takes" in L.tg_last_error()
        assert L.tg_call(e, None, n, None) == BAD
    assert L.tg_call(5, bytes(96), 12, None) == BAD and L.tg_call(-1, bytes(96), 12, None) == BAD
    # logits dtype stride B V u t k p m token lp
    ok = [4096, 1, 100, 2, 100, 64, 64, 0, 0, 0, 64, 0]
    for i, v, st in ((3, 70000, BAD), (3, 2 ** 32 + 1, BAD), (4, 2 ** 33, BAD), (4, 2 ** 19 + 1, BAD), (0, 4097, ALIGN), (1, 2, BAD)):
        a = list(ok)
        a[i] = v
        assert L.tg_call(4, struct.pack("<12q", *a), 12, None) == st, (i, v)
    w = _write(D=64)[:-1]
    assert L.tg_call(0, struct.pack("<15q", *w), 15, None) == NO
    assert L.tg_call(0, struct.pack("<15q", *_write(start=4)[:-1]), 15, None) == BAD
    a = [4096, 0, 128, 0, 0, 16384, 64, 0, 0, 0, 64, 5, 6, 0, 4096, 0, 128, 0, 0, 1, 4, 2, 128, float("nan")]
    assert L.tg_call(3, struct.pack("<23qd", *a), 24, None) == BAD and b"softmax_scale" in L.tg_last_error()


def test_workspace_is_asked_of_the_cache_device(monkeypatch):
    """Devices of different SM counts: each one's own size, whichever is current."""
    current = [0]

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.was

    class Lib:
        @staticmethod
        def tg_decode_attn_kv4_workspace(B, Hq, Hkv, n_keys, out):
            out._obj.value = 1000 + current[0]
            return 0

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_lib, "lib", lambda: Lib)
    ops._kv4_workspace.cache_clear()
    try:
        for cur in (0, 1):
            current[0] = cur
            assert [ops._kv4_workspace(i, 1, 16, 8, 9000) for i in (0, 1, 0)] == [1000, 1001, 1000]
    finally:
        ops._kv4_workspace.cache_clear()


def test_a_copied_cache_is_its_own():
    """What the calls get of a copied or unpickled cache is its own tensor's address, not the original's."""
    import copy
    import pickle
    c = object.__new__(KV4Cache)
    c.batch, c.capacity, c.n_kv_heads = 1, 40, 2
    c.data, c.bf16 = torch.zeros(1, 2, 2, 4608, dtype=torch.uint8), torch.empty(0, dtype=torch.bfloat16)
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert d.data.data_ptr() != c.data.data_ptr()
        assert d.ptr == d.data.data_ptr() and d.index == -1 and (d.batch, d.capacity, d.n_kv_heads) == (1, 40, 2)
    c.data = torch.zeros(1, 2, 2, 4608, dtype=torch.uint8)
    assert c.ptr == c.data.data_ptr()


def test_imports_on_a_torch_without_cuda():
    """The package and the calls' bindings on a torch that lacks the private functions of a CUDA build."""
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "for n in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "import tokengate_b200\n"
            "from tokengate_b200 import _lib, ops, kv4, decode\n"
            "_lib._bind_torch()\n"
            "assert _lib._get_device is torch.cuda.current_device and callable(_lib._raw_stream)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def _model_of(Hq=16, Hkv=8, head_dim=128, vocab=1000):
    from types import SimpleNamespace as NS
    w = torch.empty(vocab, 8, device="meta")
    cfg = NS(num_attention_heads=Hq, num_key_value_heads=Hkv, head_dim=head_dim, hidden_size=Hq * 128)
    return NS(config=cfg, parameters=lambda: iter([torch.empty(1)]), lm_head=NS(weight=w), model=NS(layers=[1, 2]))


def test_generation_is_refused_before_the_prefill(monkeypatch):
    """What the 4-bit cache or the sampler does not serve, and settings that do not fit the batch."""
    from tokengate_b200 import decode

    class Ran(Exception):
        pass

    def prefill(*a, **k):
        raise Ran

    monkeypatch.setattr(decode, "prefill_batch_for_decode", prefill)

    def go(model, n=3, **kw):
        return decode.generate_batch(model, None, [[1, 2, 3]] * 2, [0, 0], [2, 2], 0, 1, n, **kw)

    for kw in (dict(head_dim=64), dict(Hq=18, Hkv=2), dict(Hq=9, Hkv=2), dict(head_dim=None, Hq=16, Hkv=1)):
        with pytest.raises(ValueError, match="kv_bits=4"):
            go(_model_of(**kw), kv_bits=4)
        with pytest.raises(Ran):                       # no decode step, no cache
            go(_model_of(**kw), n=1, kv_bits=4)
        with pytest.raises(Ran):
            go(_model_of(**kw))
    for kw in (dict(), dict(Hq=8, Hkv=8), dict(Hq=24, Hkv=3), dict(head_dim=None)):
        with pytest.raises(Ran):
            go(_model_of(**kw), kv_bits=4)
    S = decode.Sampling
    for s in (S(temperature=[1.0, 1.0, 1.0]), S(temperature=None), S(top_p=float("nan")), S(top_k=[5])):
        with pytest.raises(ValueError):
            go(_model_of(), sampling=s)
    with pytest.raises(ValueError, match="vocabular"):
        go(_model_of(vocab=(1 << 19) + 1), sampling=S())
    with pytest.raises(Ran):
        go(_model_of(vocab=1 << 19), sampling=S(temperature=[0.5, 1.0], top_k=3))


@pytest.mark.parametrize("k", [0.5, 2.7, float("nan"), float("inf"), 2 ** 40, -2 ** 33])
def test_top_k_is_a_whole_number(k):
    """Not cut to one: 0.5 would turn the rule off."""
    from tokengate_b200.decode import Sampling
    with pytest.raises(ValueError):
        Sampling(top_k=k).on(1, "cpu")
    with pytest.raises(ValueError):
        Sampling(top_k=[3, k]).on(2, "cpu")
    with pytest.raises(ValueError):
        ops._per_row("top_k", k, 1, torch.int32, -1)
    assert Sampling(top_k=[3.0, 7.0]).on(2, "cpu")["top_k"].tolist() == [3, 7]
    assert Sampling(top_k=-1).on(2, "cpu")["top_k"].dtype == torch.int32


def test_decode_cache_releases_each_layer(monkeypatch):
    """When a layer is quantised, the bf16 K/V of the layers before it are gone."""
    import weakref
    from types import SimpleNamespace as NS
    from tokengate_b200 import decode
    fused = [torch.zeros(1, 5, 8, 128, dtype=torch.bfloat16) for _ in range(3)]     # one projection per layer, K/V its views
    held = [weakref.ref(t) for t in fused]
    layers = [NS(k_tok=t[:, :, 4:6], v_tok=t[:, :, 6:]) for t in fused]
    del fused
    alive = []

    def write(c, k, v):
        alive.append([i for i, r in enumerate(held) if r() is not None or layers[i].k_tok is not None])
        assert k.shape == v.shape == (1, 5, 2, 128) and c == (1, 9, 2)

    monkeypatch.setattr(decode, "KV4Cache", lambda B, n, H, device: (B, n, H))
    monkeypatch.setattr(ops, "kv4_write", write)
    dc = decode._DecodeCacheKV4(NS(layers=layers), 3, 4)
    assert alive == [[0, 1, 2], [1, 2], [2]] and dc.width == [5, 5, 5] and len(dc.kv) == 3


def test_no_cpu_path():
    with pytest.raises(ValueError, match="CUDA"):
        KV4Cache(1, 8, 2, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_tokens(torch.zeros(1, 8), torch.zeros(1))
