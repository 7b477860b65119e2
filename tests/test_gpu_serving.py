"""The paged serving operators as a server calls them: many calls queued without waiting while the shared workspace grows,
two contexts at once in two threads, the largest and smallest sizes, rows beyond one launch."""
import threading

import numpy as np
import pytest
import torch

import soc_amd as S
from tests.device import Arrays

pytestmark = pytest.mark.gpu


class Attention:
    """One attention call's operands, and its result in 64 bits."""

    def __init__(self, ctx, mem, seed, n, longest, nq=8, nkv=2, hd=64, page=16):
        rng = np.random.default_rng(seed)
        self.ctx, self.mem, self.n, self.nq, self.nkv, self.hd, self.page = ctx, mem, n, nq, nkv, hd, page
        self.lens = rng.integers(0, longest + 1, n)
        held = -(-self.lens // page)
        self.width = max(1, int(held.max()))
        pages = int(held.sum()) + 1
        self.table = np.zeros((n, self.width), np.int32)
        order = rng.permutation(pages).astype(np.int32)
        self.table[np.arange(self.width)[None, :] < held[:, None]] = order[: held.sum()]
        self.k, self.v = (rng.standard_normal((pages, nkv, page, hd)).astype(np.float16) for _ in range(2))
        self.q = rng.standard_normal((n, nq * hd)).astype(np.float32)
        self.pk, self.pv, self.pq = mem.up(self.k), mem.up(self.v), mem.up(self.q)
        self.pt, self.pl = mem.up(self.table), mem.up(self.lens.astype(np.int32))
        self.po = mem.up(np.full_like(self.q, 9.0))
        self.cache = S.PagedCache(self.pk, self.pv, pages, page, nkv, hd)

    def queue(self):
        S.paged_attention_decode(self.ctx, self.cache, self.pq, self.nq * self.hd, "f32", self.pt, self.width, self.width,
                                 self.pl, self.n, self.nq, 0.0, self.po, self.nq * self.hd)

    def wrong(self):
        out = self.mem.down(self.po).reshape(self.n, self.nq, self.hd)
        g = self.nq // self.nkv
        worst = 0.0
        for b, length in enumerate(self.lens):
            want = np.zeros((self.nq, self.hd))
            if length:
                mine = self.table[b, : -(-length // self.page)]
                k, v = (t[mine].transpose(1, 0, 2, 3).reshape(self.nkv, -1, self.hd)[:, :length].astype(np.float64)
                        for t in (self.k, self.v))
                for h in range(self.nq):
                    s = k[h // g] @ self.q[b].reshape(self.nq, self.hd)[h].astype(np.float64) / np.sqrt(self.hd)
                    p = np.exp(s - s.max())
                    want[h] = p @ v[h // g] / p.sum()
            worst = max(worst, float(np.abs(out[b] - want).max()))
        return worst


class Logprobs:
    def __init__(self, ctx, mem, seed, rows, vocab, top=8):
        rng = np.random.default_rng(seed)
        self.ctx, self.mem, self.rows, self.vocab, self.top = ctx, mem, rows, vocab, top
        self.x = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
        self.t = rng.integers(0, vocab, rows).astype(np.int32)
        self.px, self.pt = mem.up(self.x), mem.up(self.t)
        self.lp, self.ids = mem.up(np.zeros(rows, np.float32)), mem.up(np.zeros((rows, top), np.int32))
        self.tl = mem.up(np.zeros((rows, top), np.float32))

    def queue(self):
        S.logprobs(self.ctx, self.px, "f32", self.vocab, self.rows, self.vocab, 1.0, self.pt, self.lp, None, None, self.top,
                   self.ids, self.tl)

    def wrong(self):
        lp, ids = self.mem.down(self.lp), self.mem.down(self.ids)
        x = self.x.astype(np.float64)
        want = x - x.max(1, keepdims=True)
        want -= np.log(np.exp(want).sum(1, keepdims=True))
        first = np.argsort(-x, axis=1, kind="stable")[:, : self.top]
        assert np.array_equal(ids, first)
        return float(np.abs(lp - want[np.arange(self.rows), self.t]).max())


# scores and sums of these sizes are off by 1e-5 at most (head_dim + 8 products of size 4, chains of 700 terms)
OFF = 1e-4


def test_calls_queued_while_the_workspace_grows(gpu_ctx):
    ctx = S.Context(0)
    try:
        with Arrays(ctx) as mem:
            jobs = [Attention(ctx, mem, 1, 2, 900), Logprobs(ctx, mem, 2, 1, 40000), Attention(ctx, mem, 3, 9, 3000),
                    Logprobs(ctx, mem, 4, 60, 30000), Attention(ctx, mem, 5, 1, 20000), Attention(ctx, mem, 6, 200, 300),
                    Logprobs(ctx, mem, 7, 2, 100), Attention(ctx, mem, 8, 3, 5000, nq=24, nkv=2)]
            for _ in range(3):
                for j in jobs:
                    j.queue()
            for j in jobs:
                assert j.wrong() < OFF
    finally:
        ctx.close()


def test_two_contexts_in_two_threads(gpu_ctx):
    """Each context has its own stream and workspace."""
    failures = []

    def work(seed):
        try:
            ctx = S.Context(0)
            with Arrays(ctx) as mem:
                jobs = [Attention(ctx, mem, seed, 5, 2500), Logprobs(ctx, mem, seed + 1, 20, 20000),
                        Attention(ctx, mem, seed + 2, 40, 700)]
                for _ in range(20):
                    for j in jobs:
                        j.queue()
                off = [j.wrong() for j in jobs]
                if max(off) >= OFF:
                    failures.append((seed, off))
            ctx.close()
        except Exception as e:  # reported by the main thread
            failures.append((seed, repr(e)))

    threads = [threading.Thread(target=work, args=(100 * i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_attention_of_many_sequences(gpu_ctx):
    with Arrays(gpu_ctx) as mem:
        job = Attention(gpu_ctx, mem, 11, 9000, 20, nq=2, nkv=2)
        job.queue()
        assert job.wrong() < OFF


def test_rope_of_more_rows_than_a_launch(gpu_ctx):
    rows = (1 << 20) + 5
    x = np.random.default_rng(12).standard_normal((rows, 2)).astype(np.float32)
    with Arrays(gpu_ctx) as mem:
        px, py = mem.up(x), mem.up(np.zeros_like(x))
        rope = S.Rope(gpu_ctx, 2)
        rope.apply(px, py, "f32", rows, 1, offset=7)
        got = mem.down(py).astype(np.float64)
        positions = np.arange(rows)[::-1].astype(np.int32).copy()
        rope.apply(px, py, "f32", rows, 1, positions=mem.up(positions))
        back = mem.down(py).astype(np.float64)
        rope.close()
    for y, p in ((got, 7.0 + np.arange(rows)), (back, positions.astype(np.float64))):
        a, b, c, s = x[:, 0].astype(np.float64), x[:, 1].astype(np.float64), np.cos(p), np.sin(p)
        tol = (np.abs(a) + np.abs(b)) * (8 * 2.0 ** -24 + np.abs(p) * 2.0 ** -50)
        assert (np.abs(y[:, 0] - (a * c - b * s)) <= tol).all() and (np.abs(y[:, 1] - (b * c + a * s)) <= tol).all()


def test_append_of_more_rows_than_a_launch(gpu_ctx):
    rows, page = (1 << 20) + 3, 256
    pages = rows // page + 1
    g = torch.Generator(device="cuda").manual_seed(13)
    k, v = (torch.randn((rows, 64), generator=g, device="cuda").half() for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    pk, pv = (torch.zeros((pages * page, 64), device="cuda", dtype=torch.float16) for _ in range(2))
    torch.cuda.synchronize()
    S.paged_append(gpu_ctx, S.PagedCache(pk.data_ptr(), pv.data_ptr(), pages, page, 1, 64), None, None, 0, k.data_ptr(), 64,
                   v.data_ptr(), 64, "f16", None, 0, rows, 0, None, slots.data_ptr())
    gpu_ctx.synchronize()
    at = slots.long()
    assert torch.equal(pk[at], k) and torch.equal(pv[at], v)
    rest = torch.ones(pages * page, device="cuda", dtype=torch.bool)
    rest[at] = False
    assert not pk[rest].any() and not pv[rest].any()


def test_logprobs_of_more_rows_than_a_launch(gpu_ctx):
    """Rows whose chunks' parts pass the workspace of one launch."""
    rows, vocab, top = 40000, 8200, 64
    g = torch.Generator(device="cuda").manual_seed(14)
    x = torch.randn((rows, vocab), generator=g, device="cuda").half()
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    lp, en = (torch.zeros(rows, device="cuda") for _ in range(2))
    rk = torch.zeros(rows, device="cuda", dtype=torch.int32)
    ids, tl = torch.zeros((rows, top), device="cuda", dtype=torch.int32), torch.zeros((rows, top), device="cuda")
    torch.cuda.synchronize()
    S.logprobs(gpu_ctx, x.data_ptr(), "f16", vocab, rows, vocab, 1.0, t.data_ptr(), lp.data_ptr(), rk.data_ptr(),
               en.data_ptr(), top, ids.data_ptr(), tl.data_ptr())
    gpu_ctx.synchronize()
    for at in (slice(0, 500), slice(rows // 2, rows // 2 + 500), slice(rows - 9000, rows - 8500), slice(rows - 500, rows)):
        y = x[at].double()
        want = torch.log_softmax(y, -1)
        assert (lp[at] - want.gather(1, t[at].long()[:, None])[:, 0]).abs().max() < OFF
        assert (en[at] + (want.exp() * want).sum(-1)).abs().max() < 10 * OFF
        best = torch.sort(y, dim=-1, descending=True, stable=True)
        assert torch.equal(ids[at].long(), best.indices[:, :top])
        place = (best.indices == t[at].long()[:, None]).int().argmax(-1)
        assert torch.equal(rk[at].long(), place)


def test_workspaces_of_other_operators_growing_in_between(gpu_ctx):
    """The contiguous attention's scratch, grown between the paged calls, leaves theirs alone."""
    ctx = S.Context(0)
    try:
        with Arrays(ctx) as mem:
            jobs = [Attention(ctx, mem, 21, 3, 3000), Logprobs(ctx, mem, 22, 3, 40000)]
            for nkv, cap in ((2, 600), (8, 5000), (32, 5000)):
                for j in jobs:
                    j.queue()
                plane = mem.up(np.ones((nkv, cap, 128), np.float16))
                q, out = mem.up(np.ones((nkv, 128), np.float32)), mem.up(np.zeros((nkv, 128), np.float32))
                S.attention_decode(ctx, q, plane, plane, out, cap, nkv, nkv, cap)
                held = [mem.up(np.full(1024, 55, np.int32)) for _ in range(8)]  # takes what was freed, if anything was
                for j in jobs:
                    j.queue()
                    assert j.wrong() < OFF
                for p in held:
                    assert (mem.down(p) == 55).all()
                assert np.array_equal(mem.down(out), np.ones((nkv, 128), np.float32))
    finally:
        ctx.close()
