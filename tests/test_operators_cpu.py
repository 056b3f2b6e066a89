"""Rotary frequencies, and the argument checks of the 8-bit serving operators
(kvx_rope, kvx_rope_append, kvx_attend_chunk, kvx_pages_*): no GPU needed, a
refused call returns before any device work."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

EINVAL, EUNSUPPORTED, ENOSPC = -1, -4, -6
A = 0x10000  # a non-null, aligned address that nothing dereferences


@pytest.fixture(scope="module")
def kvx():
    import kvx as k
    return k


# -------------------------------------------------------------- frequencies ---

def formula(d, base, scaling, factor, low, high, ctx):
    """(angle per position of each pair, amplitude) from the definitions."""
    if scaling == "ntk" and d > 2:
        base = base * factor ** (d / (d - 2))
    f = [base ** (-2 * i / d) for i in range(d // 2)]
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling == "llama3":
        out = []
        for x in f:
            turns = ctx * x / (2 * math.pi)
            if turns <= low:
                out.append(x / factor)
            elif turns >= high:
                out.append(x)
            else:
                m = (turns - low) / (high - low)
                out.append((1 - m) * x / factor + m * x)
        return out, 1.0
    if scaling == "yarn":
        pair = lambda n: d * math.log(ctx / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), d - 1)
        out = []
        for i, x in enumerate(f):
            r = min(max((i - first) / max(last - first, 0.001), 0), 1)
            out.append(x * (1 - r) + x / factor * r)
        return out, 0.1 * math.log(factor) + 1
    return f, 1.0


@pytest.mark.parametrize("scaling,factor,low,high", [("none", 1, 1, 4), ("linear", 4, 1, 4), ("ntk", 8, 1, 4),
                                                     ("llama3", 32, 1, 4), ("yarn", 16, 1, 32)])
@pytest.mark.parametrize("d", [2, 10, 64, 128, 1024])
def test_frequencies_follow_the_formulas(kvx, scaling, factor, low, high, d):
    turns, amplitude = kvx.rope_frequencies(d, 500000.0, scaling, factor, low, high, 8192.0)
    want, amp = formula(d, 500000.0, scaling, factor, low, high, 8192.0)
    assert len(turns) == d // 2
    for t, f in zip(turns, want):
        # a power, a few products and the quotient by 2 pi, each half a unit
        # of 2^-53 off at most but the power's (2): 16 units in all
        assert abs(t / 2.0 ** 64 - f / (2 * math.pi)) <= 16 * 2.0 ** -53 * f / (2 * math.pi) + 2.0 ** -64
    assert amplitude == pytest.approx(amp, rel=2.0 ** -24)


def test_frequencies_keep_fractions_of_fast_pairs(kvx):
    """More than a turn per position: whole turns drop out."""
    turns, _ = kvx.rope_frequencies(4, 1e-4)  # pair 1: 100 radians a position
    want = (100.0 / (2 * math.pi)) % 1.0
    assert turns[1] / 2.0 ** 64 == pytest.approx(want, abs=1e-13)


@pytest.mark.parametrize("bad", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=1026), dict(base=0.0),
                                 dict(base=float("nan")), dict(base=float("inf")), dict(scaling="linear", factor=0.5),
                                 dict(scaling="ntk", factor=float("nan")), dict(scaling="llama3", factor=2.0, low=4.0, high=4.0),
                                 dict(scaling="llama3", factor=2.0, low=0.0), dict(scaling="yarn", factor=2.0, original_context=0.0),
                                 dict(scaling="yarn", factor=2.0, base=0.5)])
def test_frequencies_refuse(kvx, bad):
    with pytest.raises(kvx.KvxError) as e:
        kvx.rope_frequencies(**{"rotary_dim": 64, **bad})
    assert e.value.status == EINVAL


# ----------------------------------------------------------------- refusals ---

def table(kvx, **kw):
    f = dict(turns=A, rotary_dim=64, layout=0, amplitude=1.0)
    f.update(kw)
    return kvx.RopeTableC(*f.values())


def rope(kvx, tab=None, positions=A, tokens=4, head_dim=128, dtype=1, num=1, inverse=0, **row):
    f = dict(in_=A, out=2 * A, heads=8, it=1024, ih=128, ot=1024, oh=128)
    f.update(row)
    rows = (kvx.RopeRows * 2)(kvx.RopeRows(*f.values()), kvx.RopeRows(*f.values()))
    return kvx.lib.kvx_rope(C.byref(tab or table(kvx)), positions, tokens, head_dim, dtype, rows, num, inverse, None)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=-1), EINVAL), (dict(head_dim=0), EINVAL), (dict(head_dim=2048), EUNSUPPORTED), (dict(dtype=2), EUNSUPPORTED),
    (dict(num=0), EINVAL), (dict(num=3), EINVAL), (dict(inverse=2), EINVAL), (dict(positions=None), EINVAL), (dict(in_=None), EINVAL),
    (dict(out=None), EINVAL), (dict(heads=-1), EINVAL), (dict(in_=A + 1), EINVAL), (dict(out=A, ot=2048), EINVAL),
    (dict(tokens=0), 0), (dict(heads=0), 0)])
def test_rope_refuses(kvx, kw, status):
    assert rope(kvx, **kw) == status


@pytest.mark.parametrize("kw", [dict(turns=None), dict(turns=A + 4), dict(rotary_dim=0), dict(rotary_dim=5), dict(rotary_dim=130),
                                dict(layout=2), dict(layout=-1)])
def test_rope_refuses_tables(kvx, kw):
    assert rope(kvx, tab=table(kvx, **kw)) == EINVAL
    assert append(kvx, tab=table(kvx, **kw)) == EINVAL


def pool(kvx, **kw):
    f = dict(pool=A, stats=A, dtype=2, num_pages=8, num_kv_heads=2, head_dim=128, page_tokens=16)
    f.update(kw)
    return kvx.KvPaged(*f.values())


def append(kvx, kv=None, bt=A, max_pages=4, q_start=A, positions=A, batch=2, total=6, tab=None, io=1, q=A, qs=1024, qo=2 * A, hq=8,
           k=A, ks=256, v=A, vs=256):
    return kvx.lib.kvx_rope_append(C.byref(kv or pool(kvx)), bt, max_pages, q_start, positions, batch, total,
                                   C.byref(tab) if tab else None, io, q, qs, qo, hq, k, ks, v, vs, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(bt=None), EINVAL), (dict(q_start=None), EINVAL), (dict(positions=None), EINVAL), (dict(batch=-1), EINVAL),
    (dict(total=-1), EINVAL), (dict(max_pages=0), EINVAL), (dict(hq=-1), EINVAL), (dict(io=2), EINVAL), (dict(io=7), EINVAL),
    (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(q=None), EINVAL), (dict(qo=None), EINVAL), (dict(ks=255), EINVAL),
    (dict(vs=128), EINVAL), (dict(qs=1016), EINVAL), (dict(ks=257), EINVAL), (dict(k=A + 8), EINVAL), (dict(v=A + 2), EINVAL),
    (dict(q=A + 4), EINVAL), (dict(qo=A, qs=2048), EINVAL), (dict(batch=0), 0), (dict(total=0), 0)])
def test_append_refuses(kvx, kw, status):
    assert append(kvx, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(pool=None), EINVAL), (dict(stats=None), EINVAL), (dict(pool=A + 8), EINVAL), (dict(stats=A + 8), EINVAL),
    (dict(dtype=5), EINVAL), (dict(num_pages=0), EINVAL), (dict(num_kv_heads=0), EINVAL), (dict(head_dim=64), EUNSUPPORTED),
    (dict(page_tokens=32), EUNSUPPORTED), (dict(dtype=0), EUNSUPPORTED)])
def test_append_refuses_pools(kvx, kw, status):
    assert append(kvx, kv=pool(kvx, **kw)) == status  # io fp16: an fp32 pool (dtype 0) takes fp32 rows only


def attend(kvx, kv=None, bt=A, max_pages=4, q_start=A, positions=A, batch=2, total=6, hq=8, q=A, out=A, io=1, causal=1, ws=A, n=None):
    if n is None:
        n = 1 << 40
    return kvx.lib.kvx_attend_chunk(C.byref(kv or pool(kvx)), bt, max_pages, q_start, positions, batch, total, hq, q, out, io, 0.0,
                                    causal, ws, n, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(bt=None), EINVAL), (dict(q_start=None), EINVAL), (dict(positions=None), EINVAL), (dict(batch=-1), EINVAL),
    (dict(total=-1), EINVAL), (dict(max_pages=0), EINVAL), (dict(hq=0), EINVAL), (dict(hq=7), EINVAL), (dict(io=2), EINVAL),
    (dict(causal=2), EINVAL), (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(q=A + 8), EINVAL), (dict(out=A + 8), EINVAL),
    (dict(ws=None), ENOSPC), (dict(n=0), ENOSPC), (dict(ws=A + 8), EINVAL), (dict(batch=0), 0), (dict(total=0), 0)])
def test_attend_refuses(kvx, kw, status):
    assert attend(kvx, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(pool=None), EINVAL), (dict(stats=None), EINVAL), (dict(pool=A + 8), EINVAL), (dict(dtype=1), EUNSUPPORTED),
    (dict(dtype=0), EUNSUPPORTED), (dict(num_pages=0), EINVAL), (dict(num_kv_heads=3), EINVAL), (dict(head_dim=64), EUNSUPPORTED),
    (dict(page_tokens=8), EUNSUPPORTED)])
def test_attend_refuses_pools(kvx, kw, status):
    assert attend(kvx, kv=pool(kvx, **kw)) == status


def test_attend_workspace_grows_and_refuses(kvx):
    f = kvx.lib.kvx_attend_chunk_workspace_bytes
    assert f(0, 1, 8, 2, 4) == f(1, 0, 8, 2, 4) == f(1, 1, 7, 2, 4) == f(1, 1, 8, 0, 4) == f(1, 1, 8, 2, 0) == 0
    assert 0 < f(1, 1, 8, 2, 4) <= f(1, 1, 8, 2, 4096)
    assert f(4, 64, 8, 2, 64) <= f(8, 64, 8, 2, 64)


# -------------------------------------------------------------------- pages ---

def books(**kw):
    from kvx.pages import PagesC
    f = dict(refcounts=A, block_table=A, seq_lens=A, num_pages=8, num_rows=4, max_pages=4)
    f.update(kw)
    return PagesC(*f.values())


@pytest.mark.parametrize("kw,status", [
    (dict(refcounts=None), EINVAL), (dict(block_table=None), EINVAL), (dict(seq_lens=None), EINVAL), (dict(num_pages=0), EINVAL),
    (dict(num_rows=0), EINVAL), (dict(max_pages=0), EINVAL), (dict(refcounts=A + 2), EINVAL),
    (dict(num_rows=1 << 20, max_pages=1 << 20), EUNSUPPORTED)])
def test_pages_refuse_tables(kvx, kw, status):
    import kvx.pages  # noqa: F401
    p, kv, big = C.byref(books(**kw)), C.byref(pool(kvx)), 1 << 40
    assert kvx.lib.kvx_pages_reserve(p, A, A, big, None, None) == status
    assert kvx.lib.kvx_pages_fork(p, kv, 1, A, A, 1, A, big, None, None) == status
    assert kvx.lib.kvx_pages_free(p, A, 1, None, None) == status
    assert kvx.lib.kvx_pages_compact(p, kv, 1, A, big, None, None, None) == status


@pytest.mark.parametrize("kw", [dict(num_pages=2 ** 31 - 1), dict(num_pages=2 ** 31 - 20000), dict(num_rows=1, max_pages=2 ** 31 - 1),
                                dict(num_rows=2 ** 31 - 1, max_pages=1)])
def test_pages_refuse_sizes_next_to_the_largest_int(kvx, kw):
    """A step past the end of such an array would not fit an int."""
    import kvx.pages  # noqa: F401
    p, kv, big = C.byref(books(**kw)), C.byref(pool(kvx, num_pages=kw.get("num_pages", 8))), 1 << 60
    assert kvx.lib.kvx_pages_reserve(p, A, A, big, None, None) == EUNSUPPORTED
    assert kvx.lib.kvx_pages_fork(p, kv, 1, A, A, 1, A, big, None, None) == EUNSUPPORTED
    assert kvx.lib.kvx_pages_free(p, A, 1, None, None) == EUNSUPPORTED
    assert kvx.lib.kvx_pages_compact(p, kv, 1, A, big, None, None, None) == EUNSUPPORTED
    assert kvx.lib.kvx_pages_free(C.byref(books()), A, 2 ** 31 - 1, None, None) == EUNSUPPORTED


def test_pages_keep_their_tensors(kvx):
    """The calls hold addresses: in-place writes go through, another tensor in
    the place of one is refused."""
    from kvx.pages import Pages
    pages = object.__new__(Pages)
    for name in ("refcounts", "block_table", "seq_lens"):
        setattr(pages, "_" + name, torch.zeros(3, dtype=torch.int32))
        t = getattr(pages, name)
        exec(f"pages.{name} += 2")
        assert getattr(pages, name) is t and t.tolist() == [2, 2, 2]
        for other in (t + 1, t.clone(), t[:], None):
            with pytest.raises(AttributeError):
                setattr(pages, name, other)
        with pytest.raises(AttributeError):
            delattr(pages, name)
        assert getattr(pages, name) is t
    pages._pools, pages._stats = (torch.zeros(1),), None
    for name in ("pools", "stats"):
        with pytest.raises(AttributeError):
            setattr(pages, name, (torch.zeros(1),))


@pytest.mark.parametrize("turns,rotary_dim,layout", [
    (torch.zeros(32, dtype=torch.int64), 128, "half"), (torch.zeros(65, dtype=torch.int64), 128, "half"),
    (torch.zeros(64, dtype=torch.int32), 128, "half"), (torch.zeros(128, dtype=torch.int64)[::2], 128, "half"),
    (torch.zeros(64, 1, dtype=torch.int64), 128, "half"), (torch.zeros(64, dtype=torch.int64), 129, "half"),
    (torch.zeros(0, dtype=torch.int64), 0, "half"), (torch.zeros(64, dtype=torch.int64), 128, "other")])
def test_rope_table_refuses(kvx, turns, rotary_dim, layout):
    """The kernels read rotary_dim / 2 turns, whatever the tensor holds."""
    with pytest.raises(ValueError):
        kvx.RopeTable(turns, rotary_dim, layout, 1.0)


def test_rope_table_keeps_its_values(kvx):
    """Its C form is made once: an attribute that is replaced would not reach
    the calls, and the turns in use would be freed."""
    t = kvx.RopeTable(torch.zeros(64, dtype=torch.int64), 128, "half", 1.0)
    for name, other in (("turns", torch.ones(64, dtype=torch.int64)), ("rotary_dim", 64), ("layout", "interleaved"), ("amplitude", 2.0)):
        with pytest.raises(AttributeError):
            setattr(t, name, other)
    t.turns += 5
    assert t.turns.data_ptr() == t.c.turns and t.c.rotary_dim == t.rotary_dim == 128 and t.c.amplitude == t.amplitude == 1.0


def test_pages_refuse_arguments(kvx):
    import kvx.pages  # noqa: F401
    L, p, kv, big = kvx.lib, C.byref(books()), C.byref(pool(kvx)), 1 << 40
    need = L.kvx_pages_workspace_bytes(8, 4)
    assert need > 0 and L.kvx_pages_workspace_bytes(0, 4) == L.kvx_pages_workspace_bytes(8, 0) == 0
    assert L.kvx_pages_reserve(p, None, A, big, None, None) == EINVAL
    assert L.kvx_pages_reserve(p, A, None, big, None, None) == ENOSPC
    assert L.kvx_pages_reserve(p, A, A, 16, None, None) == ENOSPC
    assert L.kvx_pages_reserve(p, A, A + 8, big, None, None) == EINVAL
    assert L.kvx_pages_fork(p, None, 1, A, A, 1, A, big, None, None) == EINVAL
    assert L.kvx_pages_fork(p, kv, 0, A, A, 1, A, big, None, None) == EINVAL
    assert L.kvx_pages_fork(p, kv, 1, A, A, -1, A, big, None, None) == EINVAL
    assert L.kvx_pages_fork(p, kv, 1, A, A, 5, A, big, None, None) == EINVAL  # more children than rows
    assert L.kvx_pages_fork(p, kv, 1, None, A, 1, A, big, None, None) == EINVAL
    assert L.kvx_pages_fork(p, kv, 1, A, A, 0, A, big, None, None) == 0
    assert L.kvx_pages_fork(p, kv, 1, A, A, 1, A, 16, None, None) == ENOSPC
    assert L.kvx_pages_free(p, None, 1, None, None) == EINVAL
    assert L.kvx_pages_free(p, A, -1, None, None) == EINVAL
    assert L.kvx_pages_free(p, A, 0, None, None) == 0
    assert L.kvx_pages_compact(p, kv, 1, A, 16, None, None, None) == ENOSPC
    assert L.kvx_pages_copy(kv, 1, None, A, 1, None, None) == EINVAL
    assert L.kvx_pages_copy(kv, 1, A, A, -1, None, None) == EINVAL
    assert L.kvx_pages_copy(kv, 1, A, A, 0, None, None) == 0


@pytest.mark.parametrize("kw", [dict(pool=None), dict(pool=A + 8), dict(stats=None), dict(dtype=9), dict(num_pages=9),
                                dict(num_kv_heads=3), dict(head_dim=64)])
def test_pages_refuse_layers(kvx, kw):
    """A layer that is unlike the first one (or the table), or incomplete."""
    import kvx.pages  # noqa: F401
    layers = (kvx.KvPaged * 2)(pool(kvx), pool(kvx, **kw))
    p = C.byref(books())
    assert kvx.lib.kvx_pages_compact(p, layers, 2, A, 1 << 40, None, None, None) == EINVAL
    assert kvx.lib.kvx_pages_fork(p, layers, 2, A, A, 1, A, 1 << 40, None, None) == EINVAL
    assert kvx.lib.kvx_pages_copy(layers, 2, A, A, 1, None, None) == EINVAL
    swapped = (kvx.KvPaged * 1)(pool(kvx, num_pages=9))
    assert kvx.lib.kvx_pages_fork(p, swapped, 1, A, A, 1, A, 1 << 40, None, None) == EINVAL


def test_host_tensors_are_refused(kvx):
    x = torch.zeros(4, 2, 128, dtype=torch.float16)
    tab = kvx.RopeTable(torch.zeros(64, dtype=torch.int64), 128, "half", 1.0)
    with pytest.raises(ValueError):
        kvx.rope(x, None, torch.zeros(4, dtype=torch.int32), tab)
    with pytest.raises(ValueError):
        kvx.rope(x, None, torch.zeros(4, dtype=torch.int64), tab)
    with pytest.raises(ValueError):
        kvx.rope(x, None, torch.zeros(3, dtype=torch.int32), tab)
    with pytest.raises(ValueError):
        kvx.rope(x.transpose(1, 2), None, torch.zeros(4, dtype=torch.int32), tab)
    with pytest.raises(ValueError):
        kvx.rope_table(64, layout="other", device="cpu")
    with pytest.raises(ValueError):
        kvx.rope_table(64, scaling="other", device="cpu")


def test_rope_does_not_lose_gradients(kvx):
    """Recorded operations end here, so a tensor whose gradient is recorded is
    refused; without recording it is a tensor like any other."""
    x, y = (torch.zeros(4, 2, 128, dtype=torch.float16) for _ in range(2))
    y.requires_grad_()
    tab = kvx.RopeTable(torch.zeros(64, dtype=torch.int64), 128, "half", 1.0)
    pos = torch.zeros(4, dtype=torch.int32)
    for args in ((y, None), (x, y), (y * 2, x)):
        with pytest.raises(ValueError, match="no_grad"):
            kvx.rope(*args, pos, tab)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):  # the next check
            kvx.rope(*args, pos, tab)
