"""A captured decode loop that runs out of pages: a sequence that a step does not serve keeps
what it holds and goes on when pages are there again.  lens is 0 for it, so the next step's past is
lens where that is above 0 and the step's own past elsewhere (a seat of no sequence, past
below 0, stays one too)."""
import numpy as np
import pytest

import pagedref

torch = pytest.importorskip("torch")

F32, F16 = 0, 1


def following(lens, past):
    return [a if a > 0 else b for a, b in zip(lens, past)]


def simulate(next_past, steps):
    """Pages that nobody holds and that are not on the list after `steps` decode steps of the plain form."""
    page, n_pages, past, new = 16, 9, [14, 30, 45, 3], [1] * 4
    free, n_free, table = np.arange(n_pages), n_pages, np.zeros((4, 8), np.int64)
    table, n_free = pagedref.plan([0] * 4, past, table, free, n_free, sum(past), page)[:2]
    for _ in range(steps):
        table, n_free, lens = pagedref.plan(past, new, table, free, n_free, 4, page)[:3]
        past = next_past(lens.tolist(), past)
    return n_pages - n_free - sum(pagedref.pages_of(max(x, 0), page) for x in past), past


def test_a_loop_over_lens_alone_would_lose_pages():
    lost, past = simulate(following, 60)
    assert lost == 0 and all(x % 16 == 0 for x in past)  # each stands where its pages end
    assert simulate(lambda lens, past: lens, 60)[0] != 0


@pytest.mark.gpu
@pytest.mark.parametrize("t,kv,group,hd,page", [(F16, 2, 4, 128, 16), (F32, 1, 3, 256, 16), (F16, 1, 8, 128, 32)])
def test_a_captured_loop_past_the_last_page(t, kv, group, hd, page):
    from test_gpu_paged_attn import dev, host
    from test_gpu_paged_chain import Server
    n = 6
    start = [page - 2, 2 * page, 3 * page - 5, 3, 0, 40]
    pages = sum(pagedref.pages_of(x, page) for x in start) + 4
    sv = Server(t, kv, group, hd, page, pages, n, 256)
    sv.other = 0
    set_ = lambda x, v: x.copy_(dev(np.int32(v)))
    past, new = [0] * n, start
    set_(sv.past, past)
    set_(sv.new, new)
    sv.feed(sum(new))
    sv.step(sum(new))
    sv.check(past, new, True)
    past = list(start)
    past[4] = -1  # a seat of no sequence
    set_(sv.past, past)
    new = [1] * n
    set_(sv.new, new)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        sv.step(n, 1)
        sv.past.copy_(torch.where(sv.lens > 0, sv.lens, sv.past))
    free = pages - sum(pagedref.pages_of(max(x, 0), page) for x in past)
    unserved = 0
    for i in range(4 * page):
        need = [pagedref.pages_of(a + 1, page) - pagedref.pages_of(a, page) if a >= 0 else 0 for a in past]
        served = [a >= 0 and (x == 0 or sum(need[:j + 1]) <= free) for j, (a, x) in enumerate(zip(past, need))]
        free -= sum(x for x, ok in zip(need, served) if ok)
        unserved += sum(a >= 0 and not ok for a, ok in zip(past, served))
        sv.feed(n)
        g.replay()
        sv.other = sum(pagedref.pages_of(a, page) for a, ok in zip(past, served) if a >= 0 and not ok)
        sv.check(past, new, False, served)
        past = [a + 1 if ok else a for a, ok in zip(past, served)]
        assert host(sv.past).tolist() == past
        torch.zeros(1 << 16, device="cuda").add_(1)  # the program's own work between replays
        torch.cuda.synchronize()
        if i == 2 * page + 3:  # one sequence ends: those that waited go on
            assert unserved > 0
            ends = [0] * n
            ends[2] = past[2]
            ed = dev(np.int32(ends))
            sv.plan.release(n, ed.data_ptr(), None, sv.table.data_ptr(), sv.width, sv.free.data_ptr(),
                            sv.n_free.data_ptr())
            free += pagedref.pages_of(past[2], page)
            waited, past[2] = list(past), -1
            set_(sv.past, past)
    assert any(a > b for a, b in zip(past, waited) if a >= 0)
    # all of them end: every page is on the list again, once
    sv.plan.release(n, sv.past.data_ptr(), None, sv.table.data_ptr(), sv.width, sv.free.data_ptr(), sv.n_free.data_ptr())
    assert host(sv.n_free).tolist() == [pages] and sorted(host(sv.free).tolist()) == list(range(pages))
