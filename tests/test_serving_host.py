"""CPU-only checks of the rotary and paged-cache operators: refusals, sizes, argument blocks."""
import ctypes
import math

import pytest
import torch

from tests._pkg import pkg, submodule

PTR = 1 << 20


def _rotary(**kw):
    L = submodule("_lib")
    r = L.SwaRotary(PTR, PTR, 0, 0, 1, 0, 1, 32, 0, 1.0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _rotary_args(r=None, **kw):
    L = submodule("_lib")
    t = L.SwaTensor(PTR, 1 << 16, 1 << 12, 64)
    a = L.SwaRotaryArgs(1, 4, 2, 8, 64, L.SWA_BF16, 0, r or _rotary(), t, t, t, t)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _cache(**kw):
    L = submodule("_lib")
    c = L.SwaPagedKV(PTR, PTR, 4096, 1024, 64, 4096, 1024, 64, PTR, 4, PTR, None, PTR, PTR, 256, 64, 256, 64,
                     9, 16, 4, 2, 2, 64, L.SWA_BF16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _decode(cache=None, **kw):
    L = submodule("_lib")
    t = L.SwaPackedTensor(PTR, 512, 64)
    a = L.SwaPagedDecodeArgs(cache or _cache(), 8, 128, 4, 0.125, t, t, None, None, None, 0, 0, 1.0, PTR, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _append(cache=None, **kw):
    L = submodule("_lib")
    t = L.SwaPackedTensor(PTR, 512, 64)
    a = L.SwaPagedAppendArgs(cache or _cache(), None, 2, 4, t, t, t, t, 1, _rotary())
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _evict(cache=None, **kw):
    L = submodule("_lib")
    a = L.SwaPagedEvictArgs(cache or _cache(), 16, 16, 2, 4, PTR, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _status(name, args):
    return getattr(pkg().lib(), name)(None if args is None else ctypes.byref(args), None)


def _tensor(**kw):
    L = submodule("_lib")
    t = L.SwaTensor(PTR, 1 << 16, 1 << 12, 64)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 1), (dict(n_q_heads=0), 1), (dict(n_kv_heads=-1), 1), (dict(seq_len=-1), 1),
    (dict(head_dim=0), 1), (dict(head_dim=130), 1), (dict(head_dim=63), 1), (dict(head_dim=62), 1), (dict(dtype=5), 2),
    (dict(q=_tensor(ptr=None)), 1), (dict(q_out=_tensor(ptr=None)), 1), (dict(k_out=_tensor(ptr=None)), 1),
    (dict(q=_tensor(stride_l=-64)), 2), (dict(k=_tensor(stride_h=-64)), 2),
    (dict(r=_rotary(n_freq=33)), 1), (dict(r=_rotary(n_freq=65)), 1), (dict(r=_rotary(n_freq=-1)), 1),
    (dict(r=_rotary(n_axes=0)), 1), (dict(r=_rotary(inv_freq=None)), 1), (dict(r=_rotary(positions=None)), 1),
    (dict(r=_rotary(axis=(ctypes.c_uint8 * 64)(1))), 1), (dict(r=_rotary(pos_stride_l=-1)), 2),
    (dict(batch=0, r=_rotary(n_axes=0)), 1),
])
def test_rotary_refusals(kw, status):
    assert _status("swa_rotary", _rotary_args(**kw)) == status


def test_empty_calls_launch_nothing():
    assert _status("swa_rotary", _rotary_args(batch=0, q=_tensor(ptr=None))) == 0
    assert _status("swa_rotary", _rotary_args(seq_len=0)) == 0
    empty = _cache(batch=0, k=None, v=None, page_table=None, seq_lens=None)
    assert _status("swa_paged_append", _append(empty, n_tokens=0)) == 0
    assert _status("swa_paged_append", _append(n_tokens=0)) == 0
    assert _status("swa_paged_decode", _decode(empty)) == 0
    assert _status("swa_paged_evict", _evict(empty)) == 0
    assert _status("swa_paged_evict", _evict(keep=64)) == 0   # the table holds no more than the budget
    for name in ("swa_rotary", "swa_paged_append", "swa_paged_decode", "swa_paged_evict"):
        assert _status(name, None) == 1


CACHES = [
    (dict(batch=-1), 1), (dict(n_kv_heads=0), 1), (dict(n_pages=-1), 1), (dict(max_pages=-1), 1), (dict(page_size=0), 1),
    (dict(page_size=24), 2), (dict(head_dim=0), 1), (dict(head_dim=256), 1), (dict(head_dim=48), 2), (dict(dtype=9), 2),
    (dict(max_pages=2**27), 2), (dict(k=None), 1), (dict(v=None), 1), (dict(page_table=None), 1), (dict(seq_lens=None), 1),
    (dict(k=PTR + 8), 2), (dict(v=PTR + 2), 2), (dict(k_stride_row=60), 2), (dict(v_stride_page=-4096), 2),
    (dict(table_stride=-1), 2), (dict(w_stride_b=-1), 2), (dict(p_stride_h=-1), 2), (dict(batch=2**30), 2),
    (dict(w_stride_b=0), 1), (dict(p_stride_h=0), 1),
]


@pytest.mark.parametrize("kw,status", CACHES)
def test_cache_refusals(kw, status):
    for name, make in (("swa_paged_append", _append), ("swa_paged_decode", _decode), ("swa_paged_evict", _evict)):
        assert _status(name, make(_cache(**kw))) == status, name


def _packed(**kw):
    L = submodule("_lib")
    t = L.SwaPackedTensor(PTR, 512, 64)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("name,make,kw,status", [
    ("swa_paged_append", _append, dict(n_tokens=-1), 1), ("swa_paged_append", _append, dict(n_tokens=3), 1),
    ("swa_paged_append", _append, dict(n_q_heads=-1), 1), ("swa_paged_append", _append, dict(use_rotary=0), 1),
    ("swa_paged_append", _append, dict(k=_packed(ptr=None)), 1), ("swa_paged_append", _append, dict(q=_packed(ptr=None)), 1),
    ("swa_paged_append", _append, dict(q_out=_packed(stride_h=-1)), 1), ("swa_paged_append", _append, dict(r=_rotary(n_freq=40)), 1),
    ("swa_paged_decode", _decode, dict(n_q_heads=7), 1), ("swa_paged_decode", _decode, dict(n_q_heads=0), 1),
    ("swa_paged_decode", _decode, dict(sink_size=-1), 1), ("swa_paged_decode", _decode, dict(softmax_scale=math.nan), 1),
    ("swa_paged_decode", _decode, dict(decay=math.nan), 1), ("swa_paged_decode", _decode, dict(q=_packed(ptr=PTR + 4)), 2),
    ("swa_paged_decode", _decode, dict(q=_packed(stride_h=60)), 2), ("swa_paged_decode", _decode, dict(o=_packed(stride_t=-8)), 1),
    ("swa_paged_decode", _decode, dict(o=_packed(ptr=None)), 1), ("swa_paged_decode", _decode, dict(weights_out=PTR, wo_stride_b=-1), 2),
    ("swa_paged_decode", _decode, dict(weights_out=PTR, wo_stride_b=256), 1),
    ("swa_paged_evict", _evict, dict(keep=0), 1), ("swa_paged_evict", _evict, dict(trigger=-1), 1),
    ("swa_paged_evict", _evict, dict(sink_size=-1), 1), ("swa_paged_evict", _evict, dict(recent=-1), 1),
    ("swa_paged_evict", _evict, dict(sink_size=9, recent=8), 1), ("swa_paged_evict", _evict, dict(recent=2**31 - 1), 1),
    ("swa_paged_evict", _evict, dict(workspace=None), 5), ("swa_paged_evict", _evict, dict(workspace_bytes=8), 5),
    ("swa_paged_evict", _evict, dict(workspace=PTR + 16), 5),
])
def test_argument_refusals(name, make, kw, status):
    assert _status(name, make(**kw)) == status


def test_evict_needs_weights_and_positions():
    assert _status("swa_paged_evict", _evict(_cache(weights=None))) == 1
    assert _status("swa_paged_evict", _evict(_cache(positions=None))) == 1


def test_workspace_sizes():
    lib = pkg().lib()
    size = lambda **kw: lib.swa_paged_decode_workspace_size(ctypes.byref(_decode(**kw)))  # noqa: E731
    args = _decode(weights_out=PTR, wo_stride_b=256, wo_stride_h=64)  # two KV heads, rows of 64 slots
    need = lib.swa_paged_decode_workspace_size(ctypes.byref(args))
    assert need >= size() and need % 256 == 0 and size(n_q_heads=7) == 0
    if need:
        args.workspace = None
        assert _status("swa_paged_decode", args) == 5
        args.workspace, args.workspace_bytes = PTR, need - 1
        assert _status("swa_paged_decode", args) == 5
        args.workspace, args.workspace_bytes = PTR + 64, need
        assert _status("swa_paged_decode", args) == 5
    assert lib.swa_paged_decode_workspace_size(None) == 0 and lib.swa_paged_evict_workspace_size(None) == 0
    assert lib.swa_paged_evict_workspace_size(ctypes.byref(_evict())) > 0


def test_python_refusals_of_a_cache():
    make = pkg().PagedKVCache
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):   # CPU tensors: no CPU path exists
        make(k, k, table, lens)
    for bad in (k[0], k[:, :, :15], torch.zeros(4, 2, 16, 48, dtype=torch.bfloat16), k[:, :0]):
        with pytest.raises(ValueError):
            make(bad, bad, table, lens)
    with pytest.raises(ValueError):
        make(k, k[:3], table, lens)
    for a, b in ((k.float(), k.float()), (k, k.half())):
        with pytest.raises(TypeError):
            make(a, b, table, lens)
    with pytest.raises(TypeError):
        make(k, k, table.long(), lens)
    with pytest.raises(TypeError):
        make(k, k, table, lens, seen=lens.long())
    with pytest.raises(ValueError):
        make(k, k, table[0], lens)
    with pytest.raises(ValueError):
        make(k, k, table, lens[:1])


def test_python_refusals_of_a_rotation():
    R = submodule("rotary")
    inv = torch.ones(32)
    with pytest.raises(ValueError):   # CPU table
        R.Rotary(inv)
    with pytest.raises(ValueError):
        R.Rotary(torch.ones(65))
    with pytest.raises(ValueError):
        R.Rotary(torch.ones(4, 4))
    f = submodule("flash_attention_gpt_oss")
    q = torch.zeros(1, 4, 8, 16, dtype=torch.float16)
    with pytest.raises(ValueError):
        f.flash_swda_with_sink(q, q, q, 4, 0, rotary=object())
    with pytest.raises(ValueError):
        f.flash_swda_with_sink(q, q, q, 4, 0, positions=torch.arange(8))
    with pytest.raises(TypeError):
        R.apply_rotary(q, q, torch.arange(8), "no rotation")


def test_oracle_rotary_and_decode_against_other_forms():
    from oracle import serving_oracle as orc
    from oracle import swa_oracle as dense
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 7, 8, generator=g, dtype=torch.float64)
    inv = torch.tensor([1.0, 0.25, 0.5])
    pos = torch.randint(0, 50, (2, 7), generator=g)
    axes = [0, 1, 1]
    y = orc.rotary(x, pos, inv, axes, scale=2.0)
    # turning back gives the input, times the scale squared; lengths of pairs are kept
    assert torch.allclose(orc.rotary(y, pos, inv, axes, scale=2.0, inverse=True)[..., :6], 4 * x[..., :6])
    # scores depend on the distance of positions alone
    a, b = torch.randn(8, generator=g, dtype=torch.float64), torch.randn(8, generator=g, dtype=torch.float64)
    one = torch.tensor([[10], [3]])
    two = torch.tensor([[4], [7]])
    dot = lambda p, q: orc.rotary(a[None], p, inv, axes) @ orc.rotary(b[None], q, inv, axes).T  # noqa: E731
    assert torch.allclose(dot(one, two), dot(one + 5, two + 5))
    # the last row of the dense attention is the single token's
    q, k, v = (torch.randn(1, h, 20, 16, generator=g) for h in (4, 2, 2))
    logits = torch.randn(4, generator=g)
    for w, s in ((6, 2), (100, 0), (1, 0)):
        o, lse, p, _, _ = orc.decode(q[0, :, -1], k[0], v[0], 20, w, s)
        ref, rl = dense.forward(q, k, v, w, s)
        assert torch.allclose(o, ref[0, :, -1]) and torch.allclose(lse * math.log(2), rl[0, :, -1])
        assert torch.allclose(p.sum(1), torch.ones(4, dtype=torch.float64))
        o, lse, _, _, _ = orc.decode(q[0, :, -1], k[0], v[0], 20, w, s, logits=logits)
        ref, rl = dense.forward_sink_logits(q, k, v, w, s, logits)
        assert torch.allclose(o, ref[0, :, -1]) and torch.allclose(lse * math.log(2), rl[0, :, -1])


def test_oracle_eviction():
    from oracle import serving_oracle as orc
    w = [5.0, 1.0, math.nan, 4.0, 2.0, 2.0, 9.0, 0.0]
    # keep 4 of 8: 9 (slot 6), 5 (0), 4 (3), then the first of the two 2s (slot 4)
    assert orc.evict(w, range(8), 8, 8, 4, 0, 0) == ([1, 2], [4, 6])
    # held: the first token and the last
    assert orc.evict(w, range(8), 8, 8, 4, 2, 1) == ([2, 3], [6, 7])


def test_evict_needs_a_count_of_tokens():
    assert _status("swa_paged_evict", _evict()) == 1                 # without seen: seq_lens, which it shortens
    assert _status("swa_paged_evict", _evict(_cache(seen=PTR))) == 1  # seq_lens itself


def _bare_cache(d=64):
    """A cache object over CPU tensors, for what is refused before the library is called."""
    P = submodule("paged")
    L = submodule("_lib")
    c = P.PagedKVCache.__new__(P.PagedKVCache)
    k = torch.zeros(4, 2, 16, d, dtype=torch.bfloat16)
    c._t = (k, k, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), None, None, None)
    c._dev, c._dtype, c._b, c._hkv, c._d, c._cap = k.device, k.dtype, 3, 2, d, 32
    c._c, c._calls = _cache(batch=3, max_pages=2), L.Calls()
    return c


@pytest.mark.parametrize("shape", [(3, 16, 20), (3, 16, 63), (3, 16, 48), (3, 16, 8), (3, 16), (3, 1, 16, 64)])
def test_queries_of_another_shape_are_refused(shape):
    with pytest.raises(ValueError):
        _bare_cache().decode(torch.zeros(shape, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        _bare_cache().decode(torch.zeros(3, 16, 64, dtype=torch.float16))
