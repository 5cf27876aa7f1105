"""What answering with a language model takes each step, as cases that are timed and checked.

paged: attention of a chunk of new tokens over a paged cache, with the write of their keys and values. The tokens of all
sequences are packed: rows starts[s] to starts[s + 1] of q, k and v are the n new tokens of sequence s, the last of its
L = lengths[s] positions, so row i of them sits at p(i) = L - n + i. Key j of s lies in page table[s, j // page], place
j % page, of the pages (pages, kv_heads, page, dim); those of the new tokens are put there first. Head h reads the key head
h // (heads / kv_heads), and

    s[i, j] = cap(scale q_i . k_j) - slope_h (p(i) - j),    cap(x) = softcap tanh(x / softcap)
    out_i   = sum_j softmax_j(s[i, j]) v_j                  over the keys j <= p(i);

rows behind the last sequence are zeros.

sample: a token for each row of logits from a given uniform number u. With weights w_j = exp((x_j - max x) / temperature) and
the order of x descending, equal ones by index: the first top_k are kept, of those the ones before which less than top_p of
their mass lies, of those the ones with w >= min_p; the token is the first whose mass with all kept before it passes
u times the kept mass, and with it comes the logarithm of its share of that mass. Temperature 0 takes the first of the order
(and keeps it alone).

int8: a linear layer whose weight is held in 8 bits with a scale for each output, on rows brought to 8 bits with a scale
each: s = max(max |x| / 127, 2^-126), y = (round(x / s) . w) s scale + bias.

`run` has both forms: elementary torch operations (own = False), and the framework's calls (own = True).
"""

from __future__ import annotations

import math
import random

import torch

own = False  # True: the framework's operators

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 1, "f16": 2, "bf16": 3}  # the C ABI's type codes


def _paged(name=None, dtype="bf16", chunks=0, fresh=1, singles=0, longest=64, ragged=True, heads=8, kv_heads=None, dim=64, page=16, softcap=0.0,
           alibi=False, spare=0):
    """`chunks` sequences with `fresh` new tokens each (with ragged, from half of them on), `singles` with one; up to `longest`
    live keys a sequence, from a quarter of it on; `spare` rows behind the last sequence."""
    case = dict(kind="paged", dtype=dtype, chunks=chunks, fresh=fresh, singles=singles, longest=longest, ragged=ragged, heads=heads,
                kv_heads=kv_heads or heads, dim=dim, page=page, softcap=softcap, alibi=alibi, spare=spare)
    return case if name is None else dict(name=name, **case)


def _sample(name=None, dtype="f32", rows=1, vocab=256, top_k=0, top_p=1.0, min_p=0.0, spread=2.5, greedy=0.0):
    """`spread`: the logits' standard deviation; `greedy`: the share of rows with temperature 0."""
    case = dict(kind="sample", dtype=dtype, rows=rows, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p, spread=spread, greedy=greedy)
    return case if name is None else dict(name=name, **case)


def _int8(name=None, dtype="bf16", rows=1, width=64, outputs=64, bias=False):
    case = dict(kind="int8", dtype=dtype, rows=rows, width=width, outputs=outputs, bias=bias)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # serving: one new token of each of 32 sequences of different lengths, four query heads to a key head
        _paged("paged_token", singles=32, longest=8192, heads=32, kv_heads=8, dim=128),
        # one user of the byte-level GPT (C5's heads): the smallest call
        _paged("paged_one", dtype="f16", singles=1, longest=512, heads=8, dim=64),
        # a part of a long prompt against what came before it, capped scores
        _paged("paged_chunk", chunks=1, fresh=2048, longest=16384, ragged=False, heads=32, kv_heads=8, dim=128, page=64, softcap=50.0),
        # a server's step: two prompts' parts beside 24 sequences that take one token; pages that end inside a tile, odd widths, a distance
        # penalty, and rows of a fixed batch that nobody uses
        _paged("paged_mixed", dtype="f16", chunks=2, fresh=500, singles=24, longest=3000, heads=12, kv_heads=4, dim=80, page=24, alibi=True, spare=37),
        # limn's default type: a small float32 model
        _paged("paged_f32", dtype="f32", chunks=3, fresh=20, singles=5, longest=300, heads=4, dim=64),
        # the byte-level GPT's own head (C5): 32 sequences
        _sample("sample_bytes", rows=32, vocab=256, top_k=40, top_p=0.95),
        # a server's step with the filters that are used together, a few rows taking the best token
        _sample("sample_batch", dtype="bf16", rows=64, vocab=65536, top_k=50, top_p=0.9, greedy=0.1),
        # the largest: flat rows, where many tokens are kept
        _sample("sample_large", rows=256, vocab=131072, top_p=0.95, spread=1.5),
        # one user
        _sample("sample_one", dtype="f16", rows=1, vocab=50257, top_p=0.9, min_p=0.02),
        # a prompt's tokens through a wide layer
        _int8("int8_prompt", rows=8192, width=4096, outputs=8192),
        # one token each of 16 sequences: the weight's bytes count
        _int8("int8_token", rows=16, width=4096, outputs=8192),
        # sizes that are no multiples of a tile
        _int8("int8_odd", dtype="f16", rows=1021, width=760, outputs=2279, bias=True),
    ]


def _span(rng, lo, hi, odd=0.4):
    """A size between lo and hi, even over its logarithm; a multiple of 16 but for `odd` of the draws."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return x if rng.random() < odd else min(hi, max(16, x // 16 * 16))


def draw(rng):
    kind = rng.choice(["paged", "paged", "paged", "paged", "sample", "sample", "sample", "int8", "int8", "int8"])
    if kind == "int8":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        rows, width = _span(rng, 1, 8192), _span(rng, 24, 8192)
        outputs = _span(rng, 17, max(17, min(16384, (1 << 38) // (rows * width))))
        return _int8(dtype=dtype, rows=rows, width=width, outputs=outputs, bias=rng.random() < 0.5)
    if kind == "sample":
        dtype, vocab = rng.choice(["f32", "f32", "bf16", "f16"]), _span(rng, 17, 131072)
        rows = _span(rng, 1, min(512, (1 << 25) // vocab))
        return _sample(dtype=dtype, rows=rows, vocab=vocab, top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]),
                       min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), spread=rng.choice([0.5, 1.5, 2.5, 6.0]), greedy=rng.choice([0.0, 0.0, 0.2]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5, 8])
    small = dtype == "f32"
    longest = _span(rng, 16, 8192 if small else 32768)
    room = max(1, min(64, (1 << 28) // (longest * dim * kv_heads)))  # sequences whose cache is no larger than a listed one's
    form = rng.choice(["singles", "singles", "chunks", "mixed"])
    fresh = 1
    if form != "singles":
        most = (1 << 30 if small else 1 << 36) // (longest * dim * kv_heads * group)  # multiplications of one product over all heads
        fresh = max(1, min(longest, 512 if small else 4096, rng.choice([2, 5, 16, 70, 300, 2048]), most))
        chunks = rng.randint(1, max(1, min(8, room, most // fresh)))
    return _paged(dtype=dtype, chunks=0 if form == "singles" else chunks, fresh=fresh, singles=0 if form == "chunks" else rng.randint(1, room),
                  longest=longest, ragged=rng.random() < 0.8, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 16, 24, 32, 64, 128, 256]),
                  softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3, spare=rng.choice([0, 0, 3, 37]))


# ---- inputs ----------------------------------------------------------------------------------------------


def _shape(case):
    """(rows, sequences, pages of a table's row) of a paged case."""
    sequences = case["chunks"] + case["singles"]
    return case["chunks"] * case["fresh"] + case["singles"] + case["spare"], sequences, -(-case["longest"] // case["page"])


def _inputs(case, seed):
    """Name -> torch tensor on the GPU, from the seed alone (and what a program knows on the host, as lists)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TORCH[case["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        x = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
        return x if std == 1.0 else x.mul_(std)

    def words(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype).cuda()

    if case["kind"] == "int8":
        n, d, m = case["rows"], case["width"], case["outputs"]
        # rows as a norm leaves them; weights as a trained layer's, brought to 8 bits once
        w = normal(m, d, std=d**-0.5, dtype=torch.float32)
        scales = (w.abs().amax(1) / 127).clamp(min=2.0**-126)
        got = dict(x=normal(n, d), w=torch.round(w / scales.unsqueeze(1)).to(torch.int8), scales=scales)
        if case["bias"]:
            got["bias"] = normal(m)
        return got
    if case["kind"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        got = dict(logits=normal(n, vocab, std=case["spread"]), u=torch.rand(n, generator=g, device="cuda"))
        warm = 0.5 + torch.rand(n, generator=g, device="cuda")  # each user's own temperature
        got["temperature"] = torch.where(torch.rand(n, generator=g, device="cuda") < case["greedy"], 0.0, warm)
        if case["top_k"]:
            got["top_k"] = torch.full((n,), case["top_k"], dtype=torch.int32, device="cuda")
        if case["top_p"] < 1:
            got["top_p"] = torch.full((n,), case["top_p"], device="cuda")
        if case["min_p"]:
            got["min_p"] = torch.full((n,), case["min_p"], device="cuda")
        return got
    rng = random.Random(seed)
    tokens, sequences, table_pages = _shape(case)
    h, kv, dim, page, longest = (case[n] for n in ("heads", "kv_heads", "dim", "page", "longest"))
    counts = [rng.randint(-(-case["fresh"] // 2), case["fresh"]) if case["ragged"] else case["fresh"] for _ in range(case["chunks"])] + [1] * case["singles"]
    lengths = [max(n, rng.randint(max(1, longest // 4), longest)) if case["ragged"] else longest for n in counts]
    starts = [sum(counts[:i]) for i in range(sequences + 1)]
    pages = sequences * table_pages + 1
    at = list(range(pages))
    rng.shuffle(at)  # a cache's pages go to whoever asks next
    table = [[at[s * table_pages + j] if j * page < lengths[s] else -1 for j in range(table_pages)] for s in range(sequences)]
    got = dict(q=normal(tokens, h, dim, std=4.0 if case["softcap"] else 1.0), k=normal(tokens, kv, dim), v=normal(tokens, kv, dim),
               key_pages=normal(pages, kv, page, dim), value_pages=normal(pages, kv, page, dim),
               starts=words(starts), lengths=words(lengths), table=words(table), counts=counts, live=lengths)
    if case["alibi"]:
        got["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
    return got


def prepare(case, seed):
    state = dict(case=dict(case), **_inputs(case, seed))
    if case["kind"] == "paged":  # a server's own buffers
        state["out"] = torch.empty_like(state["q"])
    elif case["kind"] == "sample":
        state["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        state["logprobs"] = torch.empty(case["rows"], device="cuda")
    else:
        state["out"] = torch.empty(case["rows"], case["outputs"], dtype=state["x"].dtype, device="cuda")
    return state


# ---- the plain forms -------------------------------------------------------------------------------------


def _plain_paged(state):
    case = state["case"]
    h, kv, dim, page, cap = (case[n] for n in ("heads", "kv_heads", "dim", "page", "softcap"))
    keys, values, out = state["key_pages"], state["value_pages"], torch.zeros_like(state["q"])
    row = 0
    for s, (n, length) in enumerate(zip(state["counts"], state["live"])):
        mine = state["table"][s, : -(-length // page)].long()
        at = torch.arange(length - n, length, device="cuda")
        where = mine[at // page]
        keys[where, :, at % page] = state["k"][row : row + n]
        values[where, :, at % page] = state["v"][row : row + n]
        k, v = (x[mine].transpose(0, 1).reshape(kv, -1, dim)[:, :length].float() for x in (keys, values))
        q = state["q"][row : row + n].float().reshape(n, kv, h // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        x = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(kv, h // kv, n, length).mul_(dim**-0.5)
        if cap:
            x = x.div_(cap).tanh_().mul_(cap)
        j = torch.arange(length, device="cuda")
        far = at.unsqueeze(1) - j
        if case["alibi"]:
            x = x.sub_(state["slopes"].reshape(kv, -1, 1, 1) * far.float())
        x = x.masked_fill_(far < 0, -math.inf)
        p = x.sub_(x.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True))
        got = torch.bmm(p.reshape(kv, -1, length), v).reshape(kv, h // kv, n, dim)
        out[row : row + n] = got.permute(2, 0, 1, 3).reshape(n, h, dim).to(out.dtype)
        row += n
    return [out, keys, values]


def _plain_sample(state):
    x = state["logits"].double()  # in 64 bits: the borders decide on tokens
    rows, vocab = x.shape
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    warm = state["temperature"].double().unsqueeze(1)
    w = ((sorted_x - sorted_x[:, :1]) / torch.where(warm > 0, warm, 1.0)).exp()
    kept = torch.ones_like(w, dtype=torch.bool)
    if "top_k" in state:
        kept = torch.arange(vocab, device="cuda") < state["top_k"].unsqueeze(1)
    w = w.where(kept, 0.0)
    before = w.cumsum(1) - w
    if "top_p" in state:
        kept = kept & (before < state["top_p"].double().unsqueeze(1) * w.sum(1, keepdim=True))
    if "min_p" in state:
        kept = kept & (w >= state["min_p"].double().unsqueeze(1))
    kept[:, 0] = True
    mass = w.where(kept, 0.0).cumsum(1)
    at = (mass <= state["u"].double().unsqueeze(1) * mass[:, -1:]).sum(1)
    at = torch.minimum(at, kept.sum(1) - 1)
    at = torch.where(warm.squeeze(1) > 0, at, 0).unsqueeze(1)
    share = torch.where(warm > 0, w.gather(1, at) / mass[:, -1:], 1.0)
    return [order.gather(1, at).squeeze(1).to(torch.int32), share.log().squeeze(1).float()]


def _plain_int8(state):
    x = state["x"].float()
    s = (x.abs().amax(1, keepdim=True) / 127).clamp(min=2.0**-126)
    y = torch.round(x / s) @ state["w"].float().t()
    y = y * s * state["scales"]
    if "bias" in state:
        y = y + state["bias"].float()
    return [y.to(state["x"].dtype)]


# ---- the framework's calls -------------------------------------------------------------------------------


def _library():
    import limn_amd.hip  # noqa: F401  (registers "hip")
    from limn_amd.seam import active_device, set_device

    try:
        return active_device().lib
    except RuntimeError:
        set_device("hip")
        return active_device().lib


def _at(state, *names):
    return [state[n].data_ptr() if n in state else None for n in names]


def _room(state, need):
    """The call's workspace, as a server keeps one."""
    if "workspace" not in state:
        state["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    return state["workspace"].data_ptr(), state["workspace"].numel(), torch.cuda.current_stream().cuda_stream


def _checked(lib, status):
    if status != 0:
        raise RuntimeError(lib.limn_hip_last_error().decode())


def _served(state):
    """A server's calls of the C ABI, on its own buffers and stream."""
    lib, case = _library(), state["case"]
    code = CODE[case["dtype"]]
    if case["kind"] == "paged":
        tokens, sequences, table_pages = _shape(case)
        h, kv, dim, page = (case[n] for n in ("heads", "kv_heads", "dim", "page"))
        sizes = [tokens, sequences, h, kv, dim, state["key_pages"].shape[0], page, table_pages]
        room = _room(state, lib.limn_hip_attend_paged_workspace(code, *sizes))
        _checked(lib, lib.limn_hip_attend_paged(*_at(state, "q", "k", "v", "key_pages", "value_pages", "starts", "lengths", "table", "slopes", "out"),
                                                code, *sizes, h * dim, kv * dim, kv * dim, dim**-0.5, case["softcap"], *room))
        return [state["out"], state["key_pages"], state["value_pages"]]
    if case["kind"] == "sample":
        sizes = [case["rows"], case["vocab"]]
        room = _room(state, lib.limn_hip_sample_workspace(code, *sizes))
        _checked(lib, lib.limn_hip_sample(*_at(state, "logits", "u", "temperature", "top_k", "top_p", "min_p", "tokens", "logprobs"), code, *sizes, case["vocab"], *room))
        return [state["tokens"], state["logprobs"]]
    sizes = [case[n] for n in ("rows", "width", "outputs")]
    room = _room(state, lib.limn_hip_int8_linear_workspace(code, *sizes))
    _checked(lib, lib.limn_hip_int8_linear(*_at(state, "x", "w", "scales", "bias", "out"), code, *sizes, *room))
    return [state["out"]]


def run(state):
    if own:
        return _served(state)
    return {"paged": _plain_paged, "sample": _plain_sample, "int8": _plain_int8}[state["case"]["kind"]](state)


# ---- the work no implementation can do without -----------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "int8":
        n, d, m = case["rows"], case["width"], case["outputs"]
        return dict(bytes=n * d * size + m * d + 4 * m + (m * size if case["bias"] else 0) + n * m * size, flops=2.0 * n * d * m)
    if case["kind"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        rules = 4 * n * (2 + bool(case["top_k"]) + (case["top_p"] < 1) + bool(case["min_p"]))
        return dict(bytes=n * vocab * size + rules + 8 * n, flops=4.0 * n * vocab)  # a difference, a weight, a sum, a comparison each
    tokens, sequences, table_pages = _shape(case)
    h, kv, dim = (case[n] for n in ("heads", "kv_heads", "dim"))
    live = 0.625 * case["longest"] if case["ragged"] else float(case["longest"])
    fresh = 0.75 * case["fresh"] if case["ragged"] else float(case["fresh"])  # expected, as the lengths are
    new = case["chunks"] * fresh + case["singles"]
    pairs = case["chunks"] * fresh * max(live - fresh / 2, fresh / 2) + case["singles"] * live
    held = 2 * (sequences * live) * kv * dim * size  # the live keys and values, the new ones (read as k and v) among them
    rows = tokens * h * dim * size + new * h * dim * size
    return dict(bytes=held + rows + 2 * new * kv * dim * size + 4 * sequences * table_pages + 8 * sequences + 4 * h * case["alibi"], flops=4.0 * h * pairs * dim)


# ---- the same values in 64 bits, from the definitions ----------------------------------------------------


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "int8":
        rows = x["x"].double()
        if rows.numel() * float(case["outputs"]) > 1e12:
            return None
        top = rows.abs().max(1, keepdim=True).values
        s = torch.maximum(top / 127.0, torch.tensor(2.0**-126, dtype=torch.float64, device="cuda"))
        y = torch.matmul(torch.round(rows / s), x["w"].double().T) * (s * x["scales"].double())
        return [y + x["bias"].double() if case["bias"] else y]
    if case["kind"] == "sample":
        got, logs = [], []
        for n in range(case["rows"]):  # one row at a time, its tokens taken by weight in the order of the definition
            z = x["logits"][n].double()
            t = float(x["temperature"][n])
            if t == 0:
                got.append(torch.nonzero(z == z.max())[0, 0])
                logs.append(z.new_zeros(()))
                continue
            order = torch.argsort(-z, stable=True)
            w = torch.exp((z[order] - z.max()) / t)
            if case["top_k"]:
                w = w[: case["top_k"]]
            end = len(w)
            if case["top_p"] < 1:
                below = torch.cumsum(w, 0) < float(x["top_p"][n]) * w.sum()  # tokens whose mass with those before falls short: the next is kept too
                end = min(end, int(below.sum()) + 1)
            if case["min_p"]:
                end = min(end, max(1, int((w >= float(x["min_p"][n])).sum())))
            mass = torch.cumsum(w[:end], 0)
            at = min(end - 1, int(torch.searchsorted(mass, x["u"][n].double() * mass[-1], right=True)))
            got.append(order[at])
            logs.append(torch.log(w[at]) - torch.log(mass[-1]))
        return [torch.stack(got).to(torch.int32), torch.stack(logs)]
    tokens, sequences, _ = _shape(case)
    h, kv, dim, page = (case[n] for n in ("heads", "kv_heads", "dim", "page"))
    if h * float(sum(x["counts"])) * case["longest"] * dim > 2e12:
        return None
    pages = [x["key_pages"].double(), x["value_pages"].double()]
    out = torch.zeros(tokens, h, dim, dtype=torch.float64, device="cuda")
    for s, (n, length) in enumerate(zip(x["counts"], x["live"])):
        first = int(x["starts"][s])
        for i in range(n):  # each new token to its place
            p = length - n + i
            for held, new in zip(pages, (x["k"], x["v"])):
                held[int(x["table"][s, p // page]), :, p % page] = new[first + i].double()
        places = torch.arange(length, device="cuda")
        of = x["table"][s].long()[places // page]
        k, v = (held[of, :, places % page] for held in pages)  # (length, kv, dim)
        hidden = places.reshape(1, -1) > torch.arange(length - n, length, device="cuda").reshape(-1, 1)
        for head in range(h):
            scores = torch.matmul(x["q"][first : first + n, head].double(), k[:, head // (h // kv)].T) / math.sqrt(dim)
            if case["softcap"]:
                scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
            if case["alibi"]:
                scores = scores - x["slopes"][head].double() * (torch.arange(length - n, length, device="cuda").reshape(-1, 1) - places)
            out[first : first + n, head] = torch.softmax(scores.masked_fill(hidden, -math.inf), 1) @ v[:, head // (h // kv)]
    return [out, *pages]
