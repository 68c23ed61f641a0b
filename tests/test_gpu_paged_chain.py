"""The paged cache as a server uses it: two layers over one plan, prompts, captured
decode steps, drafts of which a part is rejected, sequences that end and others that
take their pages; rotation by the plan's positions in front.  Attention against the
plain 64-bit form over each sequence's own K and V (tolerances of
test_gpu_paged_attn.py), pages against a count of what sequences hold."""
import numpy as np
import pytest

import pagedref
from oi import paged, rope
from test_gpu_paged_attn import F16, F32, NP, dev, host, tolerance

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {F32: torch.float32, F16: torch.float16}


class Server:
    def __init__(self, t, kv, group, hd, page, n_pages, seqs, rows_max):
        self.t, self.kv, self.h, self.hd, self.page, self.n = t, kv, kv * group, hd, page, seqs
        self.rng = np.random.default_rng(hd + page + t)
        self.plan = paged.Paged(kv, hd, n_pages, page)
        self.n_pages, self.width = n_pages, 24
        g = torch.Generator(device="cuda").manual_seed(3)
        # what was in memory before is anything
        self.bufs = [torch.randint(0, 256, (self.plan.nbytes,), dtype=torch.uint8, device="cuda", generator=g) for _ in range(2)]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.randint(-9, 9999, (seqs, self.width), generator=g, **i32)
        self.free = torch.arange(n_pages, **i32).flip(0).contiguous()
        self.n_free = torch.tensor([n_pages], **i32)
        self.past, self.new, self.lens = (torch.zeros(seqs, **i32) for _ in range(3))
        self.starts = torch.zeros(seqs + 1, **i32)
        self.slots, self.pos = torch.zeros(rows_max, **i32), torch.zeros(3 * rows_max, **i32)
        self.turn = rope.RopeAxes(self.h, kv, hd, hd, [hd // 2, 0, 0], False, 1e-6)
        self.freq = dev((1e4 ** (-np.arange(hd // 2) / (hd // 2))).astype(np.float32))
        self.norm = dev((1 + 0.1 * self.rng.standard_normal(hd)).astype(np.float32))
        f = dict(dtype=torch.float32, device="cuda")
        self.x = [[torch.zeros(rows_max, w, hd, **f) for w in (self.h, kv, kv)] for _ in range(2)]
        self.q, self.k, self.v = ([torch.zeros(rows_max, w, hd, dtype=DT[t], device="cuda") for _ in range(2)]
                                  for w in (self.h, kv, kv))
        self.out = [torch.zeros(rows_max, self.h, hd, dtype=DT[t], device="cuda") for _ in range(2)]
        need = max(self.plan.prompts_workspace_bytes(self.h, seqs, rows_max),
                   max(self.plan.tokens_workspace_bytes(self.h, seqs, n) for n in (1, 4)))
        self.ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
        # each sequence's K and V per layer, as the cache holds them
        self.held = [[[np.zeros((0, kv, hd), np.float16)] * 2 for _ in range(2)] for _ in range(seqs)]

    def step(self, rows, n_q=None):
        """The device's part of a step of `rows` packed rows: plan, then each layer."""
        st = torch.cuda.current_stream().cuda_stream
        p = lambda x: x.data_ptr()
        self.plan.plan(self.n, p(self.past), p(self.new), p(self.table), self.width, p(self.free), p(self.n_free), rows,
                       p(self.lens), p(self.starts), p(self.slots), p(self.pos), stream=st)
        for i in range(2):
            x = self.x[i]
            self.turn.launch(rows, p(self.pos), p(self.freq), p(self.norm), p(self.norm), F32, p(x[0]), p(x[1]), self.t,
                             p(self.q[i]), p(self.k[i]), stream=st)
            self.v[i][:rows].copy_(x[2][:rows])
            self.plan.append(p(self.bufs[i]), self.t, p(self.k[i]), p(self.v[i]), rows, p(self.slots), stream=st)
            if n_q is None:
                self.plan.prompts(p(self.bufs[i]), self.h, self.t, p(self.q[i]), self.n, rows, p(self.starts), p(self.lens),
                                  p(self.table), self.width, p(self.out[i]), p(self.ws), self.ws.numel(), stream=st)
            else:
                self.plan.tokens(p(self.bufs[i]), self.h, self.t, p(self.q[i]), self.n, n_q, p(self.lens), p(self.table),
                                 self.width, p(self.out[i]), p(self.ws), self.ws.numel(), stream=st)

    def feed(self, rows):
        for x in self.x:
            for y in x:
                y[:rows].copy_(dev(self.rng.standard_normal((rows,) + y.shape[1:]).astype(np.float32)))

    def check(self, past, new, prompts, served=None):
        """What a step left; past and new as the host counts them."""
        served = [True] * self.n if served is None else served
        lens, starts = host(self.lens), host(self.starts)
        assert lens.tolist() == [a + b if ok else 0 for a, b, ok in zip(past, new, served)]
        assert starts.tolist() == np.cumsum([0] + list(new)).tolist()
        pages = sum(pagedref.pages_of(int(x), self.page) for x in lens)
        assert int(host(self.n_free)[0]) == self.n_pages - pages - self.other
        used = [int(x) for i in range(self.n) for x in host(self.table)[i, :pagedref.pages_of(int(lens[i]), self.page)]]
        rest = host(self.free)[:int(host(self.n_free)[0])].tolist()
        assert len(set(used + rest)) == len(used) + len(rest), "a page belongs to two"
        for i in range(2):
            q, k, v, out = (host(x[i]) for x in (self.q, self.k, self.v, self.out))
            for s in range(self.n):
                a, b = starts[s], starts[s + 1]
                if not served[s]:
                    assert (out[a:b] == 0).all()
                    continue
                old = self.held[s][i]
                self.held[s][i] = [np.concatenate([old[j][:past[s]], pagedref.stored(x[a:b])]) for j, x in enumerate((k, v))]
                if b > a:
                    kk, vv = (x.transpose(1, 0, 2).astype(np.float64) for x in self.held[s][i])
                    want, size, top = pagedref.attention(q[a:b], kk, vv, self.hd ** -0.5)
                    tol = tolerance(size, top, int(lens[s]), self.hd, self.t, prompts)
                    assert (np.abs(out[a:b] - want) <= tol).all(), (i, s)


@pytest.mark.parametrize("t,kv,group,hd,page", [(F16, 2, 4, 128, 16), (F32, 1, 3, 128, 64), (F16, 2, 8, 256, 32), (F32, 2, 2, 256, 16)])
def test_a_server_at_work(t, kv, group, hd, page):
    n = 6
    sv = Server(t, kv, group, hd, page, 900 // page, n, 512)
    sv.other = 0
    set_ = lambda x, v: x.copy_(dev(np.int32(v)))
    # prompts of five of them, the sixth not there yet
    past, new = [0] * n, [70, 3, 129, 16, 33, 0]
    set_(sv.past, past)
    set_(sv.new, new)
    sv.feed(256)
    sv.step(256)
    sv.check(past, new, True)
    past = [a + b for a, b in zip(past, new)]
    # the sixth's prompt and a token of each of the others, packed
    new = [1, 1, 1, 1, 1, 90]
    set_(sv.past, past)
    set_(sv.new, new)
    sv.feed(100)
    sv.step(100)
    sv.check(past, new, True)
    past = [a + b for a, b in zip(past, new)]
    # decode steps: one captured graph, its lengths moved on by itself; drafts of four tokens in another
    # graph over the same workspace
    graphs = {}
    side = torch.cuda.Stream()
    for n_q in (1, 4):
        set_(sv.new, [n_q] * n)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            sv.step(n * n_q, n_q)
            sv.past.copy_(sv.lens)
        graphs[n_q] = g
    set_(sv.past, past)
    for i in range(9):
        n_q = 4 if i % 4 == 2 else 1
        new = [n_q] * n
        set_(sv.new, new)
        sv.feed(n * n_q)
        graphs[n_q].replay()
        sv.check(past, new, False)
        past = [a + b for a, b in zip(past, new)]
        if n_q == 4:  # a part of each draft is rejected
            keep = [a - (j + i) % 4 for j, a in enumerate(past)]
            kd = dev(np.int32(keep))
            sv.plan.release(n, sv.lens.data_ptr(), kd.data_ptr(), sv.table.data_ptr(), sv.width, sv.free.data_ptr(),
                            sv.n_free.data_ptr())
            past = keep
            set_(sv.past, past)
        torch.zeros(1 << 16, device="cuda").add_(1)  # the program's own work between replays
        torch.cuda.synchronize()
    # two sequences end, and a prompt that the pool could not hold before takes their place
    ends = [0] * n
    ends[2], ends[5] = past[2], past[5]
    ed = dev(np.int32(ends))
    before = int(host(sv.n_free)[0])
    sv.plan.release(n, ed.data_ptr(), None, sv.table.data_ptr(), sv.width, sv.free.data_ptr(), sv.n_free.data_ptr())
    past[2] = past[5] = 0
    assert int(host(sv.n_free)[0]) == before + pagedref.pages_of(ends[2], page) + pagedref.pages_of(ends[5], page)
    room = int(host(sv.n_free)[0]) * page
    new = [0, 1, min(room - page - 40, 300), 1, 1, 0]
    set_(sv.past, past)
    set_(sv.new, new)
    rows = sum(new)
    sv.feed(rows)
    sv.step(rows)
    sv.check(past, new, True)
    past = [a + b for a, b in zip(past, new)]
    # a sequence that the list cannot serve: nothing of it is stored, its rows come out 0, the others go on
    left = int(host(sv.n_free)[0])
    new = [1, 1, 1, 1, 1, (left + 1) * page]
    assert sum(new) <= 512
    need = [pagedref.pages_of(a + b, page) - pagedref.pages_of(a, page) for a, b in zip(past, new)]
    served = [x == 0 or sum(need[:j + 1]) <= left for j, x in enumerate(need)]
    assert not served[5] and served[0]
    set_(sv.past, past)
    set_(sv.new, new)
    sv.feed(sum(new))
    for o in sv.out:
        o.fill_(7)
    sv.step(sum(new))
    lens = host(sv.lens)
    sv.other = sum(pagedref.pages_of(a, page) for a, ok in zip(past, served) if not ok)  # held, not served
    assert lens[5] == 0
    sv.check(past, new, True, served)


def test_many_sequences():
    """More than a lane's share of them: 5000 of a token or two, and packed prompts of 4700."""
    from test_gpu_paged_attn import Batch, queries
    rng = np.random.default_rng(5)
    ends = rng.integers(0, 40, 5000).tolist()
    ends[4321], ends[77] = 900, 0
    b = Batch(5, 1, 128, 16, ends)
    for t, n_q in ((F32, 1), (F16, 2)):
        q = queries(rng, 5000 * n_q, 2, 128, t)
        b.check(b.tokens(2, t, n_q, q), q, [i * n_q for i in range(5001)], t, False, 128 ** -0.5)
    ends = rng.integers(0, 30, 4700).tolist()
    ends[4600] = 700
    b = Batch(6, 1, 128, 16, ends)
    new = [int(rng.integers(0, min(e, 4) + 1)) for e in ends]
    new[4600] = 300
    starts = np.cumsum([0] + new).tolist()
    for t in (F32, F16):
        q = queries(rng, starts[-1], 2, 128, t)
        b.check(b.prompts(2, t, starts, starts[-1], q), q, starts, t, True, 128 ** -0.5)
