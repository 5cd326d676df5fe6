"""The selection operators as a program runs them: captured into CUDA graphs, on
streams, and together in the decode loop of a small model -- routed experts, beam
search, caches that follow the beams and are cut to a budget -- against the
same loop from the 64-bit definitions."""
import numpy as np
import pytest
import torch

import mflat_b200 as M
import select_ref as R

pytestmark = pytest.mark.gpu


class Ops:
    """One program's operators with results and scratch of their own."""

    def __init__(self, seed, stream=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t, e, k, b, w, v, h, cap = 700, 64, 4, 3, 4, 9001, 2, 300
        self.g, self.dims = g, (t, e, k, b, w, v, h, cap)
        self.router = M.Router(e, k, score="sigmoid", renormalise=True, groups=4, groups_kept=2, group_top=2)
        self.search = M.BeamSearch(w, v, w, dtype="bf16")
        self.cache = M.CacheEviction(h, 1, cap, 200, 32, 32, recent=10, sink=2)

        def room(n):
            return torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")

        def ints(*s):
            return torch.zeros(*s, dtype=torch.int32, device="cuda")

        self.ws = [room(self.router.workspace_bytes(t)), room(self.search.workspace_bytes(b)),
                   room(self.cache.workspace_bytes(b))]
        self.x, self.bias = torch.empty(t, e, device="cuda"), torch.empty(e, device="cuda")
        self.ids, self.w, self.start, self.slots = ints(t, k), torch.zeros(t, k, device="cuda"), ints(e + 1), ints(t * k)
        self.grad, self.dx = torch.empty(t, k, device="cuda"), torch.empty(t, e, device="cuda")
        self.logits, self.cum = torch.empty(b, w, v, dtype=torch.bfloat16, device="cuda"), torch.empty(b, w, device="cuda")
        self.parents, self.tokens, self.scores = ints(b, w), ints(b, w), torch.zeros(b, w, device="cuda")
        self.states = torch.empty(6, b, w, 40, device="cuda")
        self.lens, self.out_lens = ints(b), ints(b)
        self.acc, self.pos = torch.empty(b, h, cap, device="cuda"), ints(b, h, cap)
        self.out_acc, self.out_pos = torch.zeros(b, h, cap, device="cuda"), ints(b, h, cap)
        self.att = torch.empty(b, h, 1, cap, device="cuda")
        self.keys = torch.empty(b, h, cap, 16, dtype=torch.bfloat16, device="cuda")
        self.values = torch.empty_like(self.keys)
        self.fresh()

    def fresh(self):
        """New inputs in the same buffers."""
        for t in (self.x, self.grad, self.logits, self.states, self.keys, self.values):
            t.normal_(generator=self.g)
        self.bias.normal_(generator=self.g).mul_(0.1)
        for t in (self.acc, self.att, self.cum):
            t.uniform_(generator=self.g)
        b, cap = self.dims[3], self.dims[7]
        self.lens.copy_(torch.tensor([cap, 150, 260], dtype=torch.int32))
        self.pos.copy_(torch.arange(cap, dtype=torch.int32, device="cuda").expand_as(self.pos))

    def call(self, stream):
        t, e, k, b, w, v, h, cap = self.dims
        self.router.route_device(self.x.data_ptr(), t, self.ids.data_ptr(), self.w.data_ptr(), bias=self.bias.data_ptr(),
                                 start=self.start.data_ptr(), slots=self.slots.data_ptr(), ws=self.ws[0].data_ptr(),
                                 ws_bytes=self.ws[0].numel(), stream=stream)
        self.router.backward_device(self.x.data_ptr(), t, self.ids.data_ptr(), self.grad.data_ptr(), self.dx.data_ptr(),
                                    stream=stream)
        self.search.select_device(self.logits.data_ptr(), self.cum.data_ptr(), b, self.parents.data_ptr(),
                                  self.tokens.data_ptr(), self.scores.data_ptr(), ws=self.ws[1].data_ptr(),
                                  ws_bytes=self.ws[1].numel(), stream=stream)
        M.beam_reorder_device(self.states.data_ptr(), self.parents.data_ptr(), 6, b, w, 160, stream=stream)
        self.cache.evict_device(b, self.lens.data_ptr(), self.lens.data_ptr(), self.acc.data_ptr(), self.pos.data_ptr(),
                                self.keys.data_ptr(), self.values.data_ptr(), self.out_lens.data_ptr(),
                                out_acc=self.out_acc.data_ptr(), out_pos=self.out_pos.data_ptr(),
                                weights=self.att.data_ptr(), queries=1, ws=self.ws[2].data_ptr(),
                                ws_bytes=self.ws[2].numel(), stream=stream)

    def before(self):
        return [t.clone() for t in (self.states, self.keys, self.values)]

    def check(self, before):
        t, e, k, b, w, v, h, cap = self.dims
        ids, wt = R.route(self.x, k, "sigmoid", self.bias, None, True, 1.0, 4, 2, 2)
        np.testing.assert_array_equal(self.ids.cpu().numpy(), ids)
        np.testing.assert_allclose(self.w.cpu().numpy(), wt, rtol=3e-6)
        start, slots = R.lists(ids, e)
        np.testing.assert_array_equal(self.start.cpu().numpy(), start)
        np.testing.assert_array_equal(self.slots.cpu().numpy()[:len(slots)], slots)
        dx, size = R.route_grad(self.x, ids, self.grad, "sigmoid", True)
        assert (np.abs(self.dx.cpu().numpy() - dx) <= 1.5e-5 * size + 1e-30).all()
        parents, tokens, scores = R.beam(self.logits, self.cum, w)
        np.testing.assert_array_equal(self.parents.cpu().numpy(), parents)
        np.testing.assert_array_equal(self.tokens.cpu().numpy(), tokens)
        assert torch.equal(self.states, R.reorder(before[0], parents.tolist()))
        lens, total, source = R.evict(self.lens.tolist(), self.lens.tolist(), self.acc, self.pos.cpu().numpy(), 200, 10, 2,
                                      self.att)
        np.testing.assert_array_equal(self.out_lens.cpu().numpy(), lens)
        for (i, j), at in source.items():
            np.testing.assert_array_equal(self.out_acc.cpu().numpy()[i, j, :len(at)], total[i, j, at])
            assert torch.equal(self.keys[i, j, :len(at)], before[1][i, j, at])
            assert torch.equal(self.values[i, j, :len(at)], before[2][i, j, at])


def test_a_stream_of_its_own():
    ops, s = Ops(1), torch.cuda.Stream()
    for _ in range(3):
        ops.fresh()
        before = ops.before()
        s.wait_stream(torch.cuda.current_stream())
        ops.call(s.cuda_stream)
        s.synchronize()
        ops.check(before)


def captured(ops):
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    ops.call(s.cuda_stream)
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        ops.call(s.cuda_stream)
    return graph


def test_captured_and_replayed_on_new_inputs():
    ops = Ops(2)
    graph = captured(ops)
    for _ in range(3):
        ops.fresh()
        before = ops.before()
        graph.replay()
        torch.cuda.synchronize()
        ops.check(before)


def test_two_graphs_at_once():
    """Two programs' graphs, each with its own scratch, replayed on two streams."""
    both = [Ops(3), Ops(4)]
    graphs, streams = [captured(o) for o in both], [torch.cuda.Stream() for _ in both]
    for _ in range(4):
        before = []
        for o in both:
            o.fresh()
            before.append(o.before())
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, x in zip(both, before):
            o.check(x)


def test_calls_back_to_back_share_scratch_in_order():
    """One scratch buffer, many calls in a row on one stream: each sees its own inputs."""
    g = torch.Generator(device="cuda").manual_seed(9)
    op = M.BeamSearch(4, 20_000, 4)
    ws = torch.empty(op.workspace_bytes(2), dtype=torch.uint8, device="cuda")
    sets = []
    for _ in range(12):
        x, cum = torch.randn(2, 4, 20_000, device="cuda", generator=g), torch.rand(2, 4, device="cuda", generator=g)
        out = [torch.zeros(2, 4, dtype=d, device="cuda") for d in (torch.int32, torch.int32, torch.float32)]
        sets.append((x, cum, out))
    stream = torch.cuda.current_stream().cuda_stream
    for x, cum, out in sets:
        op.select_device(x.data_ptr(), cum.data_ptr(), 2, *(t.data_ptr() for t in out), ws=ws.data_ptr(),
                         ws_bytes=ws.numel(), stream=stream)
    torch.cuda.synchronize()
    for x, cum, out in sets:
        p, t, _ = R.beam(x, cum, 4)
        np.testing.assert_array_equal(out[0].cpu().numpy(), p)
        np.testing.assert_array_equal(out[1].cpu().numpy(), t)


# --------------------------------------------------------------- the decode loop
B, W, V, D, E, K, CAP, BUDGET = 2, 3, 211, 16, 8, 2, 24, 12


class Model:
    """One attention head over a cache per beam, one layer of routed experts, logits.
    Products in 64 bits on both sides, so that only the operators differ."""

    def __init__(self):
        g = torch.Generator().manual_seed(77)

        def mat(*s):
            return torch.randn(*s, generator=g, dtype=torch.float64)

        self.embed, self.q, self.k, self.v = mat(V, D), mat(D, D) / 2, mat(D, D) / 2, mat(D, D) / 4
        self.router, self.experts, self.head = mat(D, E), mat(E, D, D) / 4, mat(D, V) / 2

    def attend(self, tokens, step, keys, values, lens):
        """Adds the tokens' rows to the caches [B * W][CAP][D]; the mix and the weights."""
        x = self.embed[tokens.reshape(-1).long()] * (1 + 0.1 * step)
        for i in range(B * W):
            keys[i, lens[i]], values[i, lens[i]] = (x[i] @ self.k).float(), (x[i] @ self.v).float()
            lens[i] += 1
        a = torch.full((B * W, CAP), float("-inf"), dtype=torch.float64)
        for i in range(B * W):
            a[i, :lens[i]] = keys[i, :lens[i]].double() @ (x[i] @ self.q)
        a = torch.softmax(a, -1)
        mix = torch.stack([a[i, :lens[i]] @ values[i, :lens[i]].double() for i in range(B * W)])
        return x + mix, a.float()

    def mix_experts(self, x, ids, w):
        return torch.stack([x[t] + sum(float(w[t, j]) * (x[t] @ self.experts[int(e)]) for j, e in enumerate(ids[t]) if e >= 0)
                            for t in range(B * W)])


def decode(own, steps=18):
    """Tokens, parents and cache positions of every step."""
    m, n = Model(), B * W
    tokens = torch.arange(n).view(B, W)
    keys, values = torch.zeros(n, CAP, D), torch.zeros(n, CAP, D)
    acc, pos, lens = torch.zeros(n, CAP), torch.zeros(n, CAP, dtype=torch.int32), [0] * n
    cum = torch.tensor([[0.0, -1e-3, -2e-3]] * B)
    done = torch.zeros(B, W, dtype=torch.uint8)
    seen = []
    router = M.Router(E, K, renormalise=True) if own else None
    search = M.BeamSearch(W, V, W, eos=5) if own else None
    cache = M.CacheEviction(1, 1, CAP, BUDGET, D * 4, D * 4, recent=3, sink=1) if own else None
    bias = torch.linspace(-0.01, 0.01, E)
    for step in range(steps):
        for i in range(n):
            pos[i, lens[i]] = step
        x, att = m.attend(tokens, step, keys, values, lens)
        logits = (x @ m.router).float()
        if own:
            c = [t.cuda() for t in (logits, bias)]
            ids, w = torch.zeros(n, K, dtype=torch.int32).cuda(), torch.zeros(n, K).cuda()
            router.route_device(c[0].data_ptr(), n, ids.data_ptr(), w.data_ptr(), bias=c[1].data_ptr())
            ids, w = ids.cpu(), w.cpu()
        else:
            ids, w = R.route(logits, K, "softmax", bias, renormalise=True)
            w = w.astype(np.float32)
        x = m.mix_experts(x, ids, w)
        out = ((x / x.norm(dim=-1, keepdim=True)) @ m.head).float().view(B, W, V)
        if own:
            # the caches are cut to their budget, then follow the beams
            def dev(t):
                return t.cuda()
            k, v, a, p, aw = dev(keys), dev(values), dev(acc), dev(pos), dev(att)
            old = torch.tensor(lens, dtype=torch.int32).cuda()
            new, s = torch.zeros_like(old), torch.full((n,), step + 1, dtype=torch.int32).cuda()
            ws = torch.empty(max(1, cache.workspace_bytes(n)), dtype=torch.uint8).cuda()
            cache.evict_device(n, old.data_ptr(), s.data_ptr(), a.data_ptr(), p.data_ptr(), k.data_ptr(), v.data_ptr(),
                               new.data_ptr(), weights=aw.data_ptr(), queries=1, ws=ws.data_ptr(), ws_bytes=ws.numel())
            x_, c_, d_ = dev(out), dev(cum), dev(done)
            pa, to, sc = [torch.zeros(B, W, dtype=t).cuda() for t in (torch.int32, torch.int32, torch.float32)]
            wb = torch.empty(max(1, search.workspace_bytes(B)), dtype=torch.uint8).cuda()
            search.select_device(x_.data_ptr(), c_.data_ptr(), B, pa.data_ptr(), to.data_ptr(), sc.data_ptr(),
                                 finished=d_.data_ptr(), ws=wb.data_ptr(), ws_bytes=wb.numel())
            for t, row in ((k, CAP * D * 4), (v, CAP * D * 4), (a, CAP * 4), (p, CAP * 4), (new, 4), (d_, 1)):
                M.beam_reorder_device(t.data_ptr(), pa.data_ptr(), 1, B, W, row)
            keys, values, acc, pos, done = k.cpu(), v.cpu(), a.cpu(), p.cpu(), d_.cpu()
            lens, parents, tokens, cum = new.tolist(), pa.cpu(), to.cpu(), sc.cpu()
        else:
            nl, total, source = R.evict(lens, [step + 1] * n, acc[:, None], pos[:, None].numpy(), BUDGET, 3, 1,
                                        att[:, None, None])
            for (i, _), at in source.items():
                l = len(at)
                keys[i, :l], values[i, :l], pos[i, :l] = keys[i, at].clone(), values[i, at].clone(), pos[i, at].clone()
                acc[i, :l] = torch.from_numpy(total[i, 0, at])
            pa, to, sc = R.beam(out, cum, W, done.numpy(), 5)
            parents, tokens, cum = torch.from_numpy(pa), torch.from_numpy(to), torch.from_numpy(sc.astype(np.float32))
            rows = (torch.arange(B)[:, None] * W + parents).view(-1)
            keys, values, acc, pos = keys[rows], values[rows], acc[rows], pos[rows]
            lens, done = [int(nl[i]) for i in rows], done.view(-1)[rows].view(B, W)
        done = done | (tokens == 5).to(torch.uint8)
        seen.append((tokens.tolist(), parents.tolist(), [sorted(pos[i, :lens[i]].tolist()) for i in range(n)]))
    return seen, cum


def test_decode_with_routing_beams_and_a_bounded_cache():
    got, gc = decode(True)
    want, wc = decode(False)
    for step, (a, b) in enumerate(zip(got, want)):
        assert a == b, step
    assert all(len(p) == BUDGET for p in got[-1][2])
    # two roundings of fp32 a step on sums of at most 100
    np.testing.assert_allclose(gc.numpy(), wc.numpy(), atol=2 * 18 * 100 * 2.0 ** -24)
