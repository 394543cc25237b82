"""The paged cache's entry points refuse, on the host and before any device
work, what their kernels do not take. The device pointers are stand-ins that
are never dereferenced; not run where a GPU is present."""
import ctypes

import pytest

import zest_b200 as Z

try:
    import torch
    _gpu = torch.cuda.is_available()
except ImportError:
    _gpu = False

pytestmark = pytest.mark.skipif(_gpu, reason="host-only: fake device pointers")
P, ODD = 0x100000, 0x100004


def cache(k=P, v=P, type=Z.TYPE_BF16, page=64, heads=8, d=128, layers=2, pages=10, strides=None):
    s = strides or (pages * page * heads * d, page * heads * d, heads * d, d)
    return Z.KvCacheDesc(k, v, type, page, heads, d, layers, pages, *s)


def batch(n=2, T=10, max_q=5, max_kv=600, q_start=P, kv_len=P, table=P, stride=10):
    return Z.KvBatchDesc(q_start, kv_len, table, stride, T, max_q, max_kv, n)


def attn(q=P, ldq=4096, heads=32, causal=1, window=0, scale=0.1, out=P, ldo=4096, y=None, ldy=0, a=None, lda=0):
    return Z.KvAttn(q, ldq, heads, causal, window, scale, out, ldo, y, ldy, a, lda)


def new(k=P, v=P, ldk=1024, ldv=1024, q=P, ldq=4096, q_out=P, ldqo=4096, heads=32, eps=1e-6, q_norm=P, k_norm=P,
        rope=P, n_dims=128, mode=Z.ROPE_NEOX):
    return Z.KvNew(k, v, ldk, ldv, q, ldq, q_out, ldqo, heads, eps, q_norm, k_norm, rope, n_dims, mode)


def refused(rc, words):
    assert rc == -1
    msg = Z.lib().zest_last_error().decode()
    assert words in msg, msg


_alive = []


def ref(x):
    _alive.append(x)
    return None if x is None else ctypes.addressof(x)


def attend(c=None, b=None, a=None, layer=0, ws=P, size=1 << 40, err=P):
    c, b, a = c or cache(), b or batch(), a or attn()
    return Z.lib().zest_kv_attend(ref(c), layer, ref(b), ref(a), ws, size, err, None)


def append(c=None, b=None, i=None, layer=0, err=P):
    c, b, i = c or cache(), b or batch(), i or new()
    return Z.lib().zest_kv_append(ref(c), layer, ref(b), ref(i), err, None)


@pytest.mark.parametrize("call", [attend, append])
def test_caches_and_batches(call):
    for kw, words in [(dict(type=Z.TYPE_F32), "BF16 or F16"), (dict(page=48), "page_size"), (dict(page=8), "page_size"),
                      (dict(heads=0), "at least one"), (dict(d=100), "multiple of 8"), (dict(d=264), "8 to 256"),
                      (dict(d=0), "8 to 256"), (dict(pages=0), "no layers or pages"), (dict(k=0), "16-byte aligned"),
                      (dict(v=ODD), "16-byte aligned"), (dict(strides=(1 << 20, 1 << 16, 1024, 100)), "strides"),
                      (dict(strides=(1 << 20, 1 << 16, 1024, 64)), "strides"),
                      (dict(strides=(1 << 20, 0, 1024, 128)), "strides"),
                      (dict(strides=(1 << 20, -(1 << 16), 1024, 128)), "strides")]:
        refused(call(c=cache(**kw)), words)
    refused(call(layer=2), "no such layer")
    refused(call(layer=-1), "no such layer")
    for kw, words in [(dict(n=-1), "65535"), (dict(n=70000), "65535"), (dict(q_start=0), "no q_start"),
                      (dict(kv_len=0), "no q_start"), (dict(table=0), "no page table"), (dict(T=-1), "2^31"),
                      (dict(max_kv=1 << 31), "2^31")]:
        refused(call(b=batch(**kw)), words)
    refused(call(err=0), "error word")


def test_attend():
    for kw, words in [(dict(heads=12), "multiple of the kv heads"), (dict(heads=0), "multiple of the kv heads"),
                      (dict(heads=8 * 129, ldq=1 << 20, ldo=1 << 20), "128 times"), (dict(scale=0.0), "scale"),
                      (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"),
                      (dict(window=-1), "window"), (dict(window=5, causal=0), "window"), (dict(q=0), "q rows"),
                      (dict(q=ODD), "q rows"), (dict(ldq=4095), "q rows"), (dict(ldq=4100), "q rows"),
                      (dict(out=0), "no output"), (dict(ldo=4000), "output rows"), (dict(out=ODD), "output rows"),
                      (dict(y=P, ldy=100), "output rows"), (dict(a=P, lda=4100), "output rows")]:
        refused(attend(a=attn(**kw)), words)
    # a call whose keys are cut needs its workspace
    b = batch(n=1, T=1, max_q=1, max_kv=100000, stride=2000)
    need = Z.lib().zest_kv_attend_workspace(ref(cache()), ref(b), ref(attn()))
    assert need > 0
    refused(attend(b=b, size=need - 1), "workspace")
    refused(attend(b=b, ws=0), "workspace")
    refused(attend(b=b, ws=ODD), "workspace")


def test_attend_workspace():
    size = lambda **kw: Z.lib().zest_kv_attend_workspace(ref(cache()), ref(batch(**kw)), ref(attn()))
    assert size(n=0, T=0, max_q=0, max_kv=0) == 0
    assert size(n=1, T=1, max_q=1, max_kv=200) == 0
    assert size(n=1, T=1000, max_q=1000, max_kv=0) == 0
    # an m and an l and a head's values in f32 for each chunk of each row
    got = size(n=1, T=1, max_q=1, max_kv=131072, stride=2048)
    assert got > 0 and got <= 148 * 4 * 32 * (128 * 4 + 8) + 256
    refused(Z.lib().zest_kv_attend_workspace(ref(cache()), ref(batch()), ref(attn(scale=-1.0))), "scale")
    refused(Z.lib().zest_kv_attend_workspace(None, ref(batch()), ref(attn())), "no cache")


def test_append():
    for kw, words in [(dict(k=0), "k and v rows"), (dict(v=ODD), "k and v rows"), (dict(ldk=1023), "k and v rows"),
                      (dict(ldv=1000), "k and v rows"), (dict(ldq=100), "q rows"), (dict(q_out=0), "q rows"),
                      (dict(ldqo=4100), "q rows"), (dict(heads=0), "q rows"), (dict(eps=float("nan")), "eps"),
                      (dict(q_norm=ODD), "norm weights"), (dict(mode=7), "rope mode"), (dict(n_dims=0), "n_dims"),
                      (dict(n_dims=130), "n_dims"), (dict(n_dims=31), "n_dims"), (dict(rope=ODD), "rope table")]:
        refused(append(i=new(**kw)), words)


def test_page_operations():
    L = Z.lib()
    t = lambda refs=P, table=P, lens=P, seqs=4, stride=10: Z.KvTablesDesc(refs, table, lens, seqs, stride)
    c, ok = cache(), t()
    calls = {
        "grow": lambda c=c, i=ok, o=ok, n=2, a=P, b=P, e=P: L.zest_kv_grow(ref(c), ref(i), ref(o), n, a, b, e, None),
        "free": lambda c=c, i=ok, o=ok, n=2, a=P, b=P, e=P: L.zest_kv_free(ref(c), ref(i), ref(o), n, a, e, None),
        "fork": lambda c=c, i=ok, o=ok, n=2, a=P, b=P, e=P, w=P: L.zest_kv_fork(ref(c), ref(i), ref(o), n, a, b, w, e,
                                                                              None),
        "compact": lambda c=c, i=ok, o=ok, n=2, a=P, b=P, e=P, w=P: L.zest_kv_compact(ref(c), ref(i), ref(o), w, e,
                                                                                    None)}
    for name, call in calls.items():
        refused(call(c=None), "no cache")
        refused(call(c=cache(d=100)), "multiple of 8")
        refused(call(i=None), "no tables")
        refused(call(o=t(refs=0)), "no tables")
        refused(call(i=t(seqs=0), o=t(seqs=0)), "no sequences")
        refused(call(o=t(stride=11)), "differ in size")
        refused(call(e=0), "error word")
        if name in ("grow", "free", "fork"):
            refused(call(n=-1), "0 to 1024")
            refused(call(n=1025), "0 to 1024")
            refused(call(a=0), "no sequence numbers")
        if name in ("fork", "compact"):
            refused(call(w=0), "workspace")
            refused(call(w=ODD), "workspace")
    refused(calls["fork"](b=0), "no sequence numbers")
    assert L.zest_kv_pages_workspace(ref(c)) >= 4 * (1 + 3 * 10)
    refused(L.zest_kv_pages_workspace(None), "no cache")


def test_a_step_of_no_rows_is_no_call():
    """As an empty tensor comes: no pointers, and nothing to do."""
    for b in (batch(T=0, max_q=0), batch(T=0), batch(n=0, T=0, q_start=0, kv_len=0, table=0, stride=0)):
        assert attend(b=b, a=attn(q=0, ldq=0, out=0, ldo=0)) == 0
        assert append(b=b, i=new(k=0, v=0, ldk=0, ldv=0, q=0, q_out=0)) == 0
        refused(attend(b=b, a=attn(heads=12)), "multiple of the kv heads")


@pytest.mark.parametrize("call", [attend, append])
def test_counts_whose_tiles_pass_32_bits(call):
    """A sequence of 2^31 - 1 rows: its last tile's rows would be counted past 2^31."""
    for kw in (dict(T=0x7fffffff, max_q=0x7fffffff), dict(T=0x7fffffff - 4095), dict(max_kv=0x7fffffff - 4095)):
        refused(call(b=batch(**kw)), "2^31")
