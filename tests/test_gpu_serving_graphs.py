"""GPU: the serving operators on streams of their own, from several threads, and in captured graphs
that are replayed several times, alone, beside eager calls and at the same time as one another,
with every result equal to the eager one, bit for bit."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import q8_model as qm
from gpu_helpers import say
from helpers import SplitMix64
from orator_amd import asr_ops, runtime
from orator_amd import decoder_attn as da

pytestmark = pytest.mark.gpu

HQ, HKV, DH, PS, SCALE = 16, 8, 128, 16, 0.088


class Step:
    """A batch's decode step: new rows quantised into the cache, both attentions over it and a
    shared prefix over a bf16 pool, and the scores of some tokens; torch holds the buffers."""

    def __init__(self, seed, B=5, L=700, shared=330, vocab=5000):
        r = SplitMix64(seed)
        self.B, self.vocab, self.shared = B, vocab, shared
        self.pages = -(-L // PS) + 1
        table, self.n = qm.table_of(r, B, self.pages)
        table[1:, :shared // PS] = table[0, :shared // PS]
        c = qm.Cache(self.n, PS, HKV, DH, rng=r)
        gpu = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        self.kq, self.ks, self.vq, self.vs = (gpu(x) for x in (c.kq, c.ks, c.vq, c.vs))
        self.kp, self.vp = (gpu(r.normal((self.n, PS, HKV, DH))).to(torch.bfloat16) for _ in "kv")
        self.table = gpu(table)
        self.pos = gpu(np.array([L - 1 - 7 * b for b in range(B)], np.int32))
        self.q, self.k, self.v = gpu(r.normal((B, HQ, DH))), gpu(r.normal((B, 1, HKV, DH))), gpu(
            r.normal((B, 1, HKV, DH)))
        self.x, self.tok = gpu(r.normal((B, vocab), 3.0)), gpu(np.arange(B, dtype=np.int32))
        self.out = {n: torch.zeros(B, HQ, DH, device="cuda") for n in ("q8", "sq8", "sbf")}
        self.out |= {"lp": torch.zeros(B, device="cuda"), "en": torch.zeros(B, device="cuda"),
                     "ids": torch.zeros(B, 6, dtype=torch.int32, device="cuda"),
                     "top": torch.zeros(B, 6, device="cuda"),
                     "k": torch.zeros(B, 40, HKV, DH, device="cuda"),
                     "v": torch.zeros(B, 40, HKV, DH, device="cuda")}
        self.zero = torch.zeros(B, dtype=torch.int32, device="cuda")

    def run(self, stream):
        p = lambda t: t.data_ptr()  # noqa: E731
        cache = [p(x) for x in (self.kq, self.ks, self.vq, self.vs)]
        paging = (p(self.table), self.pages, PS, self.n)
        tail = (self.B, HQ, HKV, DH, SCALE, stream)
        da.WriteKvCacheQ8Paged(p(self.k), p(self.v), HKV * DH, *cache, *paging, self.B, 1, HKV, DH,
                               p(self.pos), stream)
        da.GqaDecodeAttnQ8Paged(p(self.q), *cache, *paging, p(self.pos), p(self.out["q8"]), *tail)
        da.GqaDecodeAttnSharedQ8Paged(p(self.q), *cache, *paging, p(self.pos), self.shared,
                                      p(self.out["sq8"]), *tail)
        da.GqaDecodeAttnSharedPaged(p(self.q), p(self.kp), p(self.vp), *paging, p(self.pos),
                                    self.shared, p(self.out["sbf"]), *tail)
        da.ReadKvCacheQ8Paged(*cache, *paging, p(self.out["k"]), p(self.out["v"]), False, self.B, 40,
                              HKV, DH, p(self.zero), stream)
        asr_ops.TokenLogprobs(p(self.x), self.vocab, p(self.tok), self.B, self.vocab, 6,
                              p(self.out["lp"]), p(self.out["en"]), p(self.out["ids"]),
                              p(self.out["top"]), stream)

    def eager(self):
        self.wipe()  # rows that are left as they were are the same everywhere
        torch.cuda.synchronize()
        self.run(None)
        torch.cuda.synchronize()
        return {n: t.clone() for n, t in self.out.items()}

    def wipe(self):
        for t in self.out.values():
            t.fill_(-1)

    def check(self, want):
        for n, t in self.out.items():
            assert torch.equal(t, want[n]), n


def capture(step, stream):
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        step.run(stream.cuda_stream)
    return g


def test_captured_and_replayed_beside_eager_work():
    step = Step(1)
    want = step.eager()
    side = torch.cuda.Stream()
    say("graph capture")
    g = capture(step, side)
    for _ in range(4):
        step.wipe()
        g.replay()
        torch.cuda.synchronize()
        step.check(want)
        step.wipe()
        step.run(None)
        torch.cuda.synchronize()
        step.check(want)
    # new inputs reach the replay: nothing is kept from the capture
    step.q.mul_(-0.5)
    step.pos.sub_(33)
    want = step.eager()
    step.wipe()
    g.replay()
    torch.cuda.synchronize()
    step.check(want)


def test_two_graphs_of_one_stream_replayed_at_the_same_time():
    """Graphs captured on one stream, of different sizes, replayed on two streams with nothing
    between them, and eager calls on a third."""
    steps = [Step(2), Step(3, B=3, L=1500, shared=64, vocab=20000), Step(4, B=6, L=333, shared=200)]
    want = [s.eager() for s in steps]
    side = torch.cuda.Stream()
    say("two graphs")
    graphs = [capture(s, side) for s in steps[:2]]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for s in steps:
            s.wipe()
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            steps[2].run(streams[2].cuda_stream)
        torch.cuda.synchronize()
        for s, w in zip(steps, want):
            s.check(w)


def test_streams_and_threads_at_once():
    steps = [Step(10 + i, B=2 + i, L=200 + 300 * i, shared=100) for i in range(4)]
    want = [s.eager() for s in steps]
    errors = []

    def work(s, w):
        try:
            st = runtime.Stream()
            for _ in range(5):
                s.run(st)
            st.synchronize()
            s.check(w)
            st.close()
        except Exception as e:  # noqa: BLE001 - handed to the main thread
            errors.append(e)

    for s in steps:
        s.wipe()
    torch.cuda.synchronize()
    say("threads")
    threads = [threading.Thread(target=work, args=(s, w)) for s, w in zip(steps, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_shrinking_calls_on_one_stream():
    """Calls one after another, each smaller: what an earlier one left in the scratch stays out."""
    st = runtime.Stream()
    for i, (B, L, shared) in enumerate([(6, 2000, 900), (3, 600, 64), (2, 100, 0), (1, 5, 3)]):
        s = Step(20 + i, B=B, L=L, shared=shared) if L > 50 else Step(20 + i, B=1, L=L, shared=shared)
        want = s.eager()
        s.wipe()
        torch.cuda.synchronize()
        say("shrinking", B, L)
        s.run(st)
        st.synchronize()
        s.check(want)
    st.close()
