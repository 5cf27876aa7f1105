"""attend_paged, int8_linear and sample one behind another by their C ABI: on a stream of the caller's, and captured into
graphs that are replayed in turn with other work between, every replay against the same calls made eagerly. And sample where a top-p's
border and the draw meet many equal logits."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from conftest import DTYPES, storage_values, upload
from limn_amd.dtypes import ABI_CODE
from limn_amd.hip import runtime
from limn_amd.paged import attend_paged
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, bfloat16, capture, int32, realize, use_device
from oracle.attend import within
from oracle.serving import sample as oracle
from serving import logit_rows, paged_inputs
from test_sample_gpu import TYPES, called, check

pytestmark = pytest.mark.gpu
BF16 = ABI_CODE[bfloat16]


class Step:
    """A layer's end and a draw: attention of `counts` new tokens over a cache, a head in 8 bits, a token for each row."""

    def __init__(self, lib, seed, counts, most, heads=4, kv_heads=2, hd=64, page=16, vocab=1500):
        self.lib, rng = lib, np.random.default_rng(seed)
        tokens, seqs, table_pages = sum(counts), len(counts), -(-most // page)
        pages = seqs * table_pages + 1
        on = lambda *shape, kind=torch.bfloat16: torch.tensor(rng.standard_normal(shape), dtype=torch.float32).to(kind).cuda()  # noqa: E731
        self.q, self.k, self.v = on(tokens, heads, hd), on(tokens, kv_heads, hd), on(tokens, kv_heads, hd)
        self.pools = [on(pages, kv_heads, page, hd) for _ in range(2)]
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()
        self.lengths = torch.tensor(rng.integers(max(counts), most + 1, seqs), dtype=torch.int32).cuda()
        self.table = torch.tensor(rng.permutation(pages)[: seqs * table_pages].reshape(seqs, -1), dtype=torch.int32).cuda()
        self.w8 = torch.tensor(rng.integers(-127, 128, (vocab, heads * hd)), dtype=torch.int8).cuda()
        self.scales = torch.full((vocab,), 0.004).cuda()
        self.u, self.top_p = torch.tensor(rng.random(tokens), dtype=torch.float32).cuda(), torch.full((tokens,), 0.9).cuda()
        self.sizes = (tokens, seqs, heads, kv_heads, hd, pages, page, table_pages)
        self.wide, self.vocab = heads * hd, vocab
        self.out, self.logits = torch.empty_like(self.q), torch.empty(tokens, vocab, dtype=torch.bfloat16, device="cuda")
        self.drawn, self.logs = torch.empty(tokens, dtype=torch.int32, device="cuda"), torch.empty(tokens, device="cuda")
        need = (lib.limn_hip_attend_paged_workspace(BF16, *self.sizes), lib.limn_hip_int8_linear_workspace(BF16, tokens, self.wide, vocab), lib.limn_hip_sample_workspace(BF16, tokens, vocab))
        self.rooms = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in need]
        self.need = need

    def run(self, stream):
        p = lambda *ts: [t.data_ptr() for t in ts]  # noqa: E731
        (tokens, _, heads, kv_heads, hd, *_), lib, hds = self.sizes, self.lib, self.sizes[4]
        check_ = runtime.check_limn
        check_(lib.limn_hip_attend_paged(*p(self.q, self.k, self.v, *self.pools, self.starts, self.lengths, self.table), None, self.out.data_ptr(), BF16, *self.sizes,
                                         heads * hds, kv_heads * hds, kv_heads * hds, hd**-0.5, 0.0, self.rooms[0].data_ptr(), self.need[0], stream))
        check_(lib.limn_hip_int8_linear(*p(self.out, self.w8, self.scales), None, self.logits.data_ptr(), BF16, tokens, self.wide, self.vocab, self.rooms[1].data_ptr(), self.need[1], stream))
        check_(lib.limn_hip_sample(*p(self.logits, self.u), None, None, self.top_p.data_ptr(), None, *p(self.drawn, self.logs), BF16, tokens, self.vocab, self.vocab,
                                   self.rooms[2].data_ptr(), self.need[2], stream))

    def change(self, seed):
        """Other inputs in the same buffers."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (self.q, self.k, self.v):
            t.normal_(generator=g)
        self.u.uniform_(generator=g)
        self.lengths.copy_((self.lengths * 7 + seed) % (self.sizes[6] * self.sizes[7] - 3) + 3)
        self.table.copy_(self.table.flip(0))

    def clear(self):
        for t in (self.out, self.logits, self.drawn, self.logs):
            t.zero_()

    def results(self):
        return [t.clone() for t in (self.out, self.logits, self.drawn, self.logs, *self.pools)]


SHAPES = [((1, 1, 1), 300, 1500), ((1,) * 40, 3000, 1500), ((200, 1, 70), 700, 1500), ((1, 2, 1), 300, 40001)]


@pytest.mark.parametrize("counts,most,vocab", SHAPES, ids=["few", "parts", "tiles", "split-rows"])
def test_a_stream_of_the_callers(hipdev, counts, most, vocab):
    step = Step(hipdev.lib, 1, counts, most, vocab=vocab)
    pools = [t.clone() for t in step.pools]
    step.run(None)
    torch.cuda.synchronize()
    want = step.results()
    for t, old in zip(step.pools, pools):
        t.copy_(old)
    step.clear()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    step.run(ctypes.c_void_p(stream.cuda_stream))
    stream.synchronize()
    for a, b in zip(step.results(), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("counts,most,vocab", SHAPES, ids=["few", "parts", "tiles", "split-rows"])
def test_two_graphs_replayed_in_turn(hipdev, counts, most, vocab):
    steps = [Step(hipdev.lib, s, counts, most, vocab=vocab) for s in (1, 2)]
    stream, graphs = torch.cuda.Stream(), []
    for step in steps:
        step.run(ctypes.c_void_p(stream.cuda_stream))
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.run(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        graphs.append(graph)
    for turn in range(5):
        for step, graph in zip(steps, graphs):
            step.change(turn)
            pools = [t.clone() for t in step.pools]
            step.clear()
            graph.replay()
            got = step.results()
            for t, old in zip(step.pools, pools):
                t.copy_(old)
            step.clear()
            torch.cuda.synchronize()
            step.run(None)
            torch.cuda.synchronize()
            for a, b in zip(got, step.results()):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", [1, 4, 64])
@pytest.mark.parametrize("top_p", [0.05, 0.5, 0.9, 0.999])
def test_borders_among_equal_logits(hipdev, dtype, steps, top_p):
    """Logits of few values, some with more members than a sorted list: draws in the border's own bin, in the one beside it, in the first."""
    rng = np.random.default_rng(steps)
    rows, vocab = 48, 9000
    logits = storage_values((np.round(rng.standard_normal((rows, vocab)) * 1.5 * steps) / steps).astype(np.float32), DTYPES[dtype])
    u = np.concatenate([[0.0, 1e-7, 0.5, 1 - 2.0**-24], rng.random(rows - 4)]).astype(np.float32)
    check(hipdev, logits, u, dtype, top_p=top_p)
    check(hipdev, logits, u, dtype, top_p=top_p, min_p=0.3)
    check(hipdev, logits, u, dtype, top_p=top_p, temperature=np.geomspace(0.05, 50, rows).astype(np.float32))
    check(hipdev, logits, u, dtype, top_p=top_p, top_k=np.geomspace(1, vocab, rows).astype(np.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,apart", [(1, 28672, 0), (36, 28675, 3), (5, 30011, 0), (2, 70001, 7), (1, 300001, 0)])
def test_rows_over_workgroups(hipdev, dtype, rows, vocab, apart):
    """Every setting at once and alone, rows that end before all others among them: nothing above minus infinity, a largest one without a
    draw, infinities, equal logits, masks that leave few."""
    rng = np.random.default_rng(rows + vocab)
    logits = storage_values((rng.standard_normal((rows, vocab)) * 3).astype(np.float32), DTYPES[dtype])
    u = rng.random(rows).astype(np.float32)
    for rules in (dict(), dict(top_p=0.9), dict(top_k=40), dict(top_k=3000), dict(min_p=0.1), dict(temperature=0.8, top_k=100, top_p=0.9, min_p=0.01), dict(top_p=0.8, min_p=0.2),
                  dict(top_p=0.8, min_p=1.5), dict(temperature=40.0, top_p=0.5)):
        check(hipdev, logits, u, dtype, apart, **rules)
    mixed = logits.copy()
    for r in range(rows):
        if r % 5 == 0:
            mixed[r] = [-np.inf, np.nan, 1.0][r // 5 % 3]
        elif r % 5 == 1:
            mixed[r, [7, vocab - 1]] = np.inf
        elif r % 5 == 2:
            mixed[r, 3:-2] = -np.inf
        elif r % 5 == 3:
            mixed[r] = np.round(mixed[r])
    warm = np.where(np.arange(rows) % 4 == 3, 0.0, 0.9).astype(np.float32)
    for rules in (dict(), dict(top_p=0.9), dict(top_k=50), dict(top_k=2, top_p=0.5)):
        check(hipdev, mixed, u, dtype, apart, temperature=warm, **rules)


def test_the_largest_vocabulary(hipdev):
    """2^24 logits. Their masses are off by sqrt(2^24) half units of 2^-38 of the largest weight, 4e-9 of it; a drawn token's is
    some 1e-3 of it, so a border moves past one in a case of 10^5."""
    rng = np.random.default_rng(3)
    logits, u = (rng.standard_normal((1, 1 << 24)) * 2.5).astype(np.float32), np.array([0.37], np.float32)
    check(hipdev, logits, u, "float32", top_p=0.8)
    with pytest.raises(NotImplementedError):
        called(hipdev, np.zeros((1, (1 << 24) + 1), np.float32), u, "float32")


def test_split_rows_captured_through_the_tensor_api(hipdev):
    """The workspace that a replay holds is the device's own, and other calls use it between two replays."""
    use_device(hipdev)
    logits, u, rng = logit_rows(7, 6, 40001, "bfloat16")
    t = Tensor.from_node(upload(hipdev, logits, DTYPES["bfloat16"]))

    def step(x, u):
        got = sample(x, u, temperature=0.8, top_p=0.9) + sample(x, u, top_k=30)
        realize(*got)
        return got

    run, full = capture(step), lambda value, kind=np.float32: np.full(6, value, kind)
    for turn in range(6):
        u = rng.random(6).astype(np.float32)
        got = run(t, Tensor(u).realize())
        for (tokens, logs), rules in ((got[:2], dict(temperature=full(0.8), top_p=full(0.9))), (got[2:], dict(top_k=full(30, np.int32)))):
            want, (lp, bound) = oracle(logits, u, **rules)
            np.testing.assert_array_equal(tokens.numpy(), want)
            within(logs.numpy(), lp, bound, "logprob")
        sample(t, Tensor(1 - u), top_p=0.5)[0].numpy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,hd", [((1, 1, 1), (40, 9, 300), 8, 2, 64), ((1,), (5,), 3, 1, 33), ((130, 2), (200, 64), 4, 4, 80), ((2, 5), (9, 70), 2, 2, 200)])
def test_queries_keys_and_values_in_one(hipdev, dtype, counts, lengths, heads, kv_heads, hd):
    """The bits of the call with each apart, through the Tensor API, captured too."""
    use_device(hipdev)
    x = paged_inputs(3, dtype=dtype, counts=counts, lengths=lengths, heads=heads, kv_heads=kv_heads, hd=hd, page=16, spare=1)
    t = DTYPES[dtype]
    on = lambda a, kind=t: Tensor.from_node(upload(hipdev, a, kind))  # noqa: E731
    where = [on(x[n], int32) for n in ("starts", "lengths", "table")]
    apart, one = ([on(x[n]) for n in ("key_pages", "value_pages")] for _ in range(2))
    together = on(np.concatenate([x[n].reshape(len(x["q"]), -1) for n in ("q", "k", "v")], 1))

    def step(qkv):
        out = attend_paged(qkv, None, None, *one, *where, softcap=5.0, heads=heads)
        realize(out)
        return out

    want = attend_paged(*(on(x[n]) for n in ("q", "k", "v")), *apart, *where, softcap=5.0).numpy()
    run = capture(step)
    for _ in range(4):
        np.testing.assert_array_equal(run(together).numpy(), want)
        for a, b in zip(one, apart):
            np.testing.assert_array_equal(a.numpy(), b.numpy())
        assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("few", [False, True], ids=["every", "few-values"])
def test_settings_of_every_split_row(hipdev, dtype, few):
    rng = np.random.default_rng(9)
    rows, vocab = 36, 30011
    logits = storage_values((rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32), DTYPES[dtype])
    if few:
        logits = np.round(logits) * rng.choice([-0.0, 0.0, 1.0], (rows, vocab)).astype(np.float32)  # both zeros are equal
    for _ in range(3):
        u = rng.choice([-1.0, 0.0, 0.3, 0.999999, 1.0, 7.0, np.nan, -1.0, 0.5], rows).astype(np.float32)
        check(hipdev, logits, u, dtype, temperature=rng.choice([-1.0, 0.0, 1e-30, 0.01, 0.5, 1.0, 2.0, 1e30, np.nan, np.inf], rows).astype(np.float32),
              top_k=rng.choice([-3, 0, 1, 2, 10, 2000, vocab - 1, vocab, 2**31 - 1], rows).astype(np.int32), top_p=rng.choice([-1.0, 0.0, 1e-9, 0.3, 0.99, 1.0, 2.0, np.nan], rows).astype(np.float32),
              min_p=rng.choice([-1.0, 0.0, 1e-9, 0.1, 1.0, 5.0, np.nan], rows).astype(np.float32))
        check(hipdev, logits, u, dtype, top_p=rng.choice([-1.0, 0.0, 1e-9, 0.3, 0.99, 1.0, 2.0, np.nan], rows).astype(np.float32), min_p=rng.choice([-1.0, 0.0, 1e-9, 0.1, 1.0, 5.0, np.nan], rows).astype(np.float32))
