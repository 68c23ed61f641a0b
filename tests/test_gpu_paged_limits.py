"""The paged cache at the ends of what its entries take: 65536 sequences, 4096 query
heads of one kv head, 1024 kv heads, a long sequence; prompts captured once and replayed
over other lengths; two calls at once.  Plain forms and tolerances of
test_gpu_paged_attn.py, pages against pagedref.py."""
import numpy as np
import pytest

import pagedref
from test_gpu_paged import State, pool
from test_gpu_paged_attn import F16, F32, Batch, dev, host, queries, tolerance

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MOST = 65536


@pytest.mark.parametrize("short", [0, 2000])
def test_plan_of_the_most_sequences(short):
    """Every thread takes 64 sequences; `short` pages fewer than they need, and a row too few."""
    rng = np.random.default_rng(short)
    past, new = rng.integers(0, 40, MOST), rng.integers(0, 3, MOST)
    need = sum(pagedref.pages_of(int(a + b), 16) - pagedref.pages_of(int(a), 16) for a, b in zip(past, new))
    n_pages = int(sum(pagedref.pages_of(int(a), 16) for a in past)) + need - short
    table, free, n_free = pool(rng, past, 16, 3, n_pages)
    s = State(table, free, n_free, n_pages, 16)
    n_rows = int(new.sum()) - (1 if short else 0)
    want = pagedref.plan(past, new, table, free, n_free, n_rows, 16)
    got = s.step(past, new, n_rows)
    assert (host(s.table) == want[0]).all() and host(s.n_free).tolist() == [want[1], 77]
    for g, w in zip(got, want[2:]):
        assert (g == w).all()
    lens, keep = dev(got[0]), dev(np.minimum(np.int32(past), got[0]))
    s.plan.release(MOST, lens.data_ptr(), keep.data_ptr(), s.table.data_ptr(), 3, s.free.data_ptr(), s.n_free.data_ptr())
    assert host(s.n_free).tolist() == [n_free, 77] and (host(s.free) == free).all()


@pytest.mark.parametrize("which,t", [("tokens", F32), ("tokens", F16), ("prompts", F32), ("prompts", F16)])
def test_attention_of_the_most_sequences(which, t):
    """64 sequences of 0 to 90 slots, each 1024 times (pages may be shared by readers), one of them long."""
    few, times = 64, MOST // 64
    rng = np.random.default_rng(4)
    ends = rng.integers(0, 91, few).tolist()
    ends[11], ends[12] = 0, 1
    b = Batch(31, 1, 128, 16, ends)
    n_q = 2
    q = queries(rng, few * n_q, 2, 128, t)
    starts = [n_q * i for i in range(few + 1)]
    want = list(b.want(q, starts, 128 ** -0.5))
    b.table_d, b.lens = b.table_d.repeat(times, 1), b.lens.repeat(times)
    b.ends = ends * times
    many = np.tile(q, (times, 1, 1))
    got = b.tokens(2, t, n_q, many) if which == "tokens" else b.prompts(2, t, [n_q * i for i in range(MOST + 1)], MOST * n_q, many)
    got = got.reshape(times, few * n_q, 2, 128).astype(np.float64)
    for i, lo, hi, (out, size, top) in want:
        tol = tolerance(size, top, ends[i], 128, t, which == "prompts")
        assert (np.abs(got[:, lo:hi] - out) <= tol).all(), i


HEADS = [  # kv heads, group, tokens of each sequence, lengths
    (1, 4096, 2, [50, 3]),
    (1, 4096, 16, [20]),
    (1024, 1, 1, [40, 7, 0]),
    (1024, 4, 3, [33]),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
@pytest.mark.parametrize("case", HEADS, ids=str)
def test_many_heads(case, which, t):
    n_kv, g, n_q, ends = case
    b = Batch(n_kv + n_q, n_kv, 128, 16, ends)
    starts = [n_q * i for i in range(len(ends) + 1)]
    q = queries(b.rng, starts[-1], n_kv * g, 128, t)
    got = b.tokens(n_kv * g, t, n_q, q) if which == "tokens" else b.prompts(n_kv * g, t, starts, starts[-1], q)
    b.check(got, q, starts, t, which == "prompts" or n_q * g > 64, 128 ** -0.5)


@pytest.mark.parametrize("t", [F32, F16])
def test_a_long_sequence_beside_none(t):
    ends = [120001, 0, 5]
    b = Batch(17, 1, 256, 64, ends)
    q = queries(b.rng, 6, 4, 256, t)
    b.check(b.tokens(4, t, 2, q), q, [0, 2, 4, 6], t, False, 256 ** -0.5)
    b.check(b.prompts(4, t, [0, 5, 5, 6], 6, q), q, [0, 5, 5, 6], t, True, 256 ** -0.5)


def test_the_largest_values():
    """Rows of f16's largest numbers: outputs end there, in each form."""
    for t in (F32, F16):
        b = Batch(23, 2, 128, 32, [300, 40])
        sign = np.where(np.arange(128) % 2, 1.0, -1.0).astype(np.float32)
        slots = np.array([int(b.table[i, j // 32]) * 32 + j % 32 for i, e in enumerate(b.ends) for j in range(e)])
        b.ref.append(np.full((340, 2, 128), 1e-3, np.float32), np.broadcast_to(1e6 * sign, (340, 2, 128)), slots)
        b.buf.copy_(dev(b.ref.buf))
        q = queries(b.rng, 8, 8, 128, t)
        for which in ("tokens", "prompts"):
            got = b.tokens(8, t, 4, q) if which == "tokens" else b.prompts(8, t, [0, 4, 8], 8, q)
            b.check(got, q, [0, 4, 8], t, which == "prompts", 128 ** -0.5, which)


@pytest.mark.parametrize("t", [F32, F16])
def test_a_captured_prompt_goes_by_the_numbers_that_it_finds(t):
    """A server's mixed step as one graph: its starts and lengths change from replay to replay."""
    lens = [[900, 130, 64, 1], [33, 2000, 0, 5], [0, 0, 0, 0], [1, 3, 260, 700]]
    news = [[100, 30, 64, 1], [33, 160, 0, 5], [0, 0, 0, 0], [1, 3, 100, 60]]
    n_rows = 200
    b = Batch(41, 2, 128, 32, [max(x) for x in zip(*lens)])
    width = b.width
    row = 8 * 128
    q = torch.zeros(n_rows, row, dtype=(torch.float32, torch.float16)[t], device="cuda")
    out = torch.zeros_like(q)
    starts = torch.zeros(5, dtype=torch.int32, device="cuda")
    need = b.plan.prompts_workspace_bytes(8, 4, n_rows)
    ws = b.workspace(need)

    def call():
        b.plan.prompts(b.buf.data_ptr(), 8, t, q.data_ptr(), 4, n_rows, starts.data_ptr(), b.lens.data_ptr(),
                       b.table_d.data_ptr(), width, out.data_ptr(), ws.data_ptr(), need,
                       stream=torch.cuda.current_stream().cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        call()
    for turn in range(8):
        i = turn % 4
        at = np.cumsum([0] + news[i])
        x = queries(b.rng, n_rows, 8, 128, t)
        q.copy_(dev(x.reshape(n_rows, row)))
        starts.copy_(dev(np.int32(at)))
        b.lens.copy_(dev(np.int32(lens[i])))
        b.ends = lens[i]
        out.fill_(7)
        g.replay()
        got = host(out).reshape(n_rows, 8, 128).copy()
        assert (got[at[-1]:] == 7).all()
        b.check(got, x, at.tolist(), t, True, 128 ** -0.5, "replay %d" % turn)
        out.fill_(7)
        call()
        assert (host(out).reshape(n_rows, 8, 128) == got).all()


def test_two_calls_at_once():
    """One cache read by two streams' calls, each with its workspace."""
    b = Batch(57, 2, 128, 64, [4000, 700, 90, 2500])
    one, two = queries(b.rng, 4, 8, 128, F16), queries(b.rng, 300, 8, 128, F16)
    at = [0, 200, 230, 240, 300]
    want = b.tokens(8, F16, 1, one), b.prompts(8, F16, at, 300, two)
    b.check(want[0], one, [0, 1, 2, 3, 4], F16, False, 128 ** -0.5)
    b.check(want[1], two, at, F16, True, 128 ** -0.5)
    q = dev(one.reshape(4, -1)), dev(two.reshape(300, -1))
    out = [torch.zeros_like(x) for x in q]
    need = b.plan.tokens_workspace_bytes(8, 4, 1), b.plan.prompts_workspace_bytes(8, 4, 300)
    ws, starts = [b.workspace(n) for n in need], dev(np.int32(at))
    st = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        b.plan.tokens(b.buf.data_ptr(), 8, F16, q[0].data_ptr(), 4, 1, b.lens.data_ptr(), b.table_d.data_ptr(), b.width,
                      out[0].data_ptr(), ws[0].data_ptr(), need[0], stream=st[0].cuda_stream)
        b.plan.prompts(b.buf.data_ptr(), 8, F16, q[1].data_ptr(), 4, 300, starts.data_ptr(), b.lens.data_ptr(),
                       b.table_d.data_ptr(), b.width, out[1].data_ptr(), ws[1].data_ptr(), need[1], stream=st[1].cuda_stream)
    for o, w in zip(out, want):
        assert (host(o).reshape(w.shape) == w).all()
