"""What the entries of the paged cache refuse before anything reaches a device, and
the sizes that they state."""
import ctypes

import pytest

from oi import _native, paged

E_ARG, E_RANGE = -1, -6
M = 1 << 26  # addresses that are never read


def lib():
    return _native.hip()


def dims(n_kv=2, hd=128, n_pages=64, page=16):
    return ctypes.byref(_native.PagedDims(n_kv, hd, n_pages, page))


def said(text):
    return text in lib().oi_last_error().decode()


@pytest.mark.parametrize("bad", [(0, 128, 4, 16), (1025, 128, 4, 16), (2, 64, 4, 16), (2, 192, 4, 16), (2, 128, 0, 16),
                                 (2, 128, 4, 8), (2, 128, 4, 128), (2, 128, 4, 48), (2, 128, (1 << 24) + 1, 16)])
def test_dims(bad):
    L = lib()
    assert L.oi_paged_bytes(dims(*bad)) == 0
    with pytest.raises(_native.OIError):
        paged.Paged(*bad)
    assert L.oi_paged_tokens_workspace_bytes(dims(*bad), 4, 1, 1) == 0
    assert L.oi_paged_prompts_workspace_bytes(dims(*bad), 4, 1, 1) == 0
    assert L.oi_paged_plan_launch(dims(*bad), 1, M, M, M, 1, M, M, 1, M, M, M, None, None) == E_ARG and said("bad dims")
    assert L.oi_paged_bytes(None) == 0


def test_bytes():
    assert paged.Paged(2, 128, 3, 16).nbytes == 2 * 2 * 3 * 16 * 128 * 2
    assert paged.Paged(8, 256, 1 << 22, 64).nbytes == 4 * 8 * 256 << 28
    p = paged.Paged(8, 128, 1000, 64)
    assert 0 < p.tokens_workspace_bytes(8, 1, 1) < p.tokens_workspace_bytes(32, 1, 1) < p.tokens_workspace_bytes(32, 1, 16)
    assert p.tokens_workspace_bytes(32, 65536, 1) == p.tokens_workspace_bytes(32, 1, 1)
    assert 0 < p.prompts_workspace_bytes(32, 1, 3) < p.prompts_workspace_bytes(32, 1, 500)
    for heads, seqs, n in [(33, 1, 1), (0, 1, 1), (32, 0, 1), (32, 65537, 1), (32, 1, 0), (8 * 1024, 1, 1)]:
        assert p.tokens_workspace_bytes(heads, seqs, n) == 0
        assert p.prompts_workspace_bytes(heads, seqs, n) == 0
    assert p.tokens_workspace_bytes(32, 1, 17) == 0
    assert p.prompts_workspace_bytes(32, 1, (1 << 24) + 1) == 0
    assert p.prompts_workspace_bytes(512, 1, 1 << 20) == 0  # group^2 * rows = 2^32


PLAN = dict(n_seqs=3, past=M, new=2 * M, table=3 * M, stride=4, free=4 * M, n_free=5 * M, rows=10, lens=6 * M, starts=7 * M,
            slots=8 * M, pos=9 * M)


def plan(**over):
    a = dict(PLAN, **over)
    return lib().oi_paged_plan_launch(dims(), a["n_seqs"], a["past"], a["new"], a["table"], a["stride"], a["free"],
                                      a["n_free"], a["rows"], a["lens"], a["starts"], a["slots"], a["pos"], None)


def test_plan_refusals():
    for over in (dict(n_seqs=0), dict(n_seqs=65537), dict(stride=0), dict(rows=-1), dict(rows=(1 << 24) + 1)):
        assert plan(**over) == E_RANGE, over
    for name in ("past", "new", "table", "free", "n_free", "lens", "starts", "slots"):
        assert plan(**{name: None}) == E_ARG and said("null"), name
        assert plan(**{name: PLAN[name] + 2}) == E_ARG and said("misaligned"), name
    # every output against every other argument, at its first and last four bytes
    size = dict(past=12, new=12, table=48, free=256, n_free=4, lens=12, starts=16, slots=40, pos=120)
    outs = ("table", "lens", "starts", "slots", "pos", "n_free")
    for o in outs:
        for other in size:
            if other != o:
                for at in (PLAN[o], PLAN[o] + size[o] - 4, PLAN[o] - size[other] + 4):
                    assert plan(**{other: at}) == E_ARG and said("overlaps"), (o, other)


def test_release_refusals():
    base = dict(n=3, held=M, keep=2 * M, table=3 * M, stride=4, free=4 * M, n_free=5 * M)

    def call(**over):
        a = dict(base, **over)
        return lib().oi_paged_release_launch(dims(), a["n"], a["held"], a["keep"], a["table"], a["stride"], a["free"],
                                             a["n_free"], None)
    assert call(n=0) == E_RANGE and call(stride=0) == E_RANGE and call(n=65537) == E_RANGE
    for name in ("held", "table", "free", "n_free"):
        assert call(**{name: None}) == E_ARG and said("null")
        assert call(**{name: base[name] + 1}) == E_ARG and said("misaligned")
    for other in ("held", "keep", "table", "n_free"):
        assert call(**{other: base["free"] + 252}) == E_ARG and said("overlaps"), other
    for other in ("held", "keep", "table"):
        assert call(**{other: base["n_free"]}) == E_ARG and said("overlaps"), other


def test_append_refusals():
    base = dict(cache=M, type=0, k=2 * M, ks=256, v=3 * M, vs=256, n=5, slots=4 * M)

    def call(**over):
        a = dict(base, **over)
        return lib().oi_paged_append_launch(dims(), a["cache"], a["type"], a["k"], a["ks"], a["v"], a["vs"], a["n"],
                                            a["slots"], None)
    for over in (dict(type=2), dict(type=8), dict(cache=None), dict(k=None), dict(v=None), dict(slots=None),
                 dict(cache=M + 128), dict(slots=4 * M + 2), dict(k=2 * M + 8), dict(v=3 * M + 4), dict(ks=255),
                 dict(vs=257), dict(ks=1 << 41)):
        assert call(**over) == E_ARG, over
    assert call(n=0) == E_RANGE and call(n=(1 << 24) + 1) == E_RANGE
    last = 2 * 2 * 64 * 16 * 128 * 2
    for over in (dict(k=M), dict(v=M + last - 16), dict(slots=M + last - 4), dict(k=M - 4 * 1024 - 16)):
        assert call(**over) == E_ARG and said("overlaps"), over


ATTN = dict(cache=M, heads=4, type=0, q=2 * M, qs=512, scale=0.1, seqs=3, n=5, starts=3 * M, lens=4 * M, table=5 * M, stride=4,
            out=6 * M, os=512, ws=8 * M, need=1 << 40)


def attn(which, **over):
    a = dict(ATTN, **over)
    L = lib()
    mid = [a["seqs"], a["n"]] + ([a["starts"]] if which == "prompts" else [])
    f = L.oi_paged_prompts_launch if which == "prompts" else L.oi_paged_tokens_launch
    return f(dims(), a["cache"], a["heads"], a["type"], a["q"], a["qs"], a["scale"], *mid, a["lens"], a["table"], a["stride"],
             a["out"], a["os"], a["ws"], a["need"], None)


@pytest.mark.parametrize("which", ["tokens", "prompts"])
def test_attention_refusals(which):
    for over in (dict(heads=3), dict(heads=0), dict(heads=4098), dict(type=2), dict(cache=None), dict(q=None), dict(out=None),
                 dict(ws=None), dict(lens=None), dict(table=None), dict(cache=M + 16), dict(ws=8 * M + 8),
                 dict(lens=4 * M + 2), dict(table=5 * M + 1), dict(q=2 * M + 8), dict(qs=510), dict(os=514),
                 dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2.5e38), dict(scale=-3.0e38)):
        assert attn(which, **over) == E_ARG, over
    for over in (dict(seqs=0), dict(seqs=65537), dict(n=0), dict(n=-1), dict(stride=0), dict(stride=(1 << 24) + 1)):
        assert attn(which, **over) == E_RANGE, over
    assert attn(which, n=17 if which == "tokens" else (1 << 24) + 1) == E_RANGE
    p = paged.Paged(2, 128, 64, 16)
    if which == "tokens":
        need = p.tokens_workspace_bytes(4, 3, 5)
    else:
        assert attn(which, starts=None) == E_ARG and attn(which, starts=3 * M + 2) == E_ARG
        need = 768 * 8  # less than any
    assert attn(which, need=need - 1) == E_ARG and said("needed")
    # out in place has q's stride; otherwise it meets nothing
    assert attn(which, out=ATTN["q"], os=516) == E_ARG and said("same stride")
    rows = 15 if which == "tokens" else 5
    for over in (dict(out=ATTN["q"] + 512), dict(out=M), dict(out=ATTN["lens"]), dict(out=ATTN["table"] + 32),
                 dict(ws=M + 256), dict(ws=ATTN["q"] + 1024), dict(ws=ATTN["lens"] - 16), dict(out=ATTN["ws"] + 64),
                 dict(out=ATTN["q"] + 512 * 4 * rows - 16)) + ((dict(out=ATTN["starts"]),) if which == "prompts" else ()):
        assert attn(which, **over) == E_ARG and said("overlaps"), over
