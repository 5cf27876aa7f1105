"""Two operators of language models, as cases that are timed and checked.

attend: attention whose scores follow rules. With p(i) = L - t_q + i the position of query i (L the live keys of its
sequence, its queries the last of them), head h reads the key head h // (heads / kv_heads), and

    s[i, j] = cap(scale q_i . k_j) - slope_h |p(i) - j|,    cap(x) = softcap tanh(x / softcap)
    out_i   = sum_j softmax_j(s[i, j]) v_j                  over the keys j that query i sees,

which are those with j < L and (j <= p(i) or j < prefix, where it is causal), of the query's own document where documents
are given (a negative document is padding: its queries see nothing, its keys are seen by none). A query that sees no key
has a row of zeros and a logsumexp of minus infinity. Trained (out, dq, dk, dv) through the Tensor API, captured once;
served (out and the logsumexp of each row) through the C ABI.

xent: the softmax cross entropy of a language model's head, from the last hidden rows and the head's weight without keeping
the logits: loss = mean over the rows with a target of logsumexp(x w^T) - (x w^T)[target], with its gradients. A negative
target leaves its row out.

`run` has both forms: elementary torch operations in 32 bits (own = False), and the framework's calls (own = True).
"""

from __future__ import annotations

import math

import torch

own = False  # True: the framework's operators

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 1, "f16": 2, "bf16": 3}  # the C ABI's type codes


def _attend(name=None, dtype="bf16", batch=1, heads=1, kv_heads=None, t_q=1, t_k=None, dim=64, causal=True, softcap=0.0, alibi=False,
            document=0, prefix=False, ragged=False, train=True):
    case = dict(kind="attend", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads or heads, t_q=t_q, t_k=t_k or t_q, dim=dim, causal=causal,
                softcap=softcap, alibi=alibi, document=document, prefix=prefix, ragged=ragged, train=train)
    return case if name is None else dict(name=name, **case)


def _xent(name=None, dtype="bf16", rows=1, width=64, vocab=256, ignored=0.0):
    case = dict(kind="xent", dtype=dtype, rows=rows, width=width, vocab=vocab, ignored=ignored)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # long-context training on packed documents (the attention of bench.py's headline, C4, with documents of some 1000 tokens)
        _attend("attend_packed", batch=8, heads=16, t_q=4096, dim=128, document=1024),
        # a layer with capped scores whose query heads share key heads
        _attend("attend_capped", batch=4, heads=16, kv_heads=4, t_q=4096, dim=128, softcap=50.0),
        # a layer of the GPT training step (C5) with the distance in place of position embeddings, on short packed texts
        _attend("attend_distance", batch=32, heads=8, t_q=512, dim=64, alibi=True, document=200),
        # training on prompts and answers: the prompt sees itself whole; ragged length, head dim 80
        _attend("attend_prefix", dtype="f16", batch=8, heads=12, kv_heads=6, t_q=1021, dim=80, prefix=True),
        # limn's default type: a small float32 model (C1) with every rule on
        _attend("attend_f32", dtype="f32", batch=2, heads=4, t_q=256, dim=64, softcap=30.0, alibi=True, document=100),
        # serving: one new token of each of 32 sequences of different lengths, four query heads to a key head
        _attend("attend_token", batch=32, heads=32, kv_heads=8, t_q=1, t_k=8192, dim=128, softcap=50.0, ragged=True, train=False),
        # serving one user: the smallest call
        _attend("attend_one_token", batch=1, heads=8, t_q=1, t_k=1000, dim=64, alibi=True, ragged=True, train=False),
        # the head of the byte-level GPT training step (C5)
        _xent("xent_bytes", rows=16384, width=512, vocab=256),
        # a large vocabulary on a batch of training tokens, part of them prompt tokens without a target
        _xent("xent_large", rows=8192, width=2048, vocab=65536, ignored=0.25),
        # a vocabulary and a width that are no multiples of a tile
        _xent("xent_odd", dtype="f16", rows=4001, width=760, vocab=50257, ignored=0.1),
        # limn's default type
        _xent("xent_f32", dtype="f32", rows=2048, width=512, vocab=8191),
        # a small batch before a large vocabulary: the weight's bytes count
        _xent("xent_few", rows=48, width=512, vocab=32000),
    ]


def _span(rng, lo, hi, odd=0.4):
    """A size between lo and hi, even over its logarithm; a multiple of 16 but for `odd` of the draws."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return x if rng.random() < odd else min(hi, max(16, x // 16 * 16))


def draw(rng):
    kind = rng.choice(["train", "train", "train", "serve", "serve", "xent", "xent", "xent"])
    if kind == "xent":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 1 << 40 if dtype != "f32" else 1 << 34  # products of one of its four matrix products
        rows, width = _span(rng, 1, 16384), _span(rng, 24, 2048)
        vocab = _span(rng, 17, max(17, min(131072, most // (rows * width))))
        return _xent(dtype=dtype, rows=rows, width=width, vocab=vocab, ignored=rng.choice([0.0, 0.0, 0.1, 0.5]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5, 8])
    rules = dict(softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.4)
    if kind == "train":
        causal = rng.random() < 0.8
        t = _span(rng, 32, 4096 if dtype != "f32" else 1024)
        most = (1 << 35) if dtype != "f32" else (1 << 30)  # multiplications of one product over all heads
        batch = max(1, min(16, most // (t * t * dim * kv_heads * group)))
        return _attend(dtype=dtype, batch=rng.randint(1, batch), heads=kv_heads * group, kv_heads=kv_heads, t_q=t, dim=dim, causal=causal,
                       document=rng.choice([0, 0, max(16, t // 8), max(16, t // 3)]), prefix=causal and rng.random() < 0.3, **rules)
    t_k = _span(rng, 16, 32768 if dtype != "f32" else 8192)
    t_q = min(t_k, rng.choice([1, 1, 1, 2, 5, 16, 70]))
    batch = max(1, min(48, (1 << 28) // (t_k * dim * kv_heads)))
    return _attend(dtype=dtype, batch=rng.randint(1, batch), heads=kv_heads * group, kv_heads=kv_heads, t_q=t_q, t_k=t_k, dim=dim, ragged=True,
                   prefix=t_q > 1 and rng.random() < 0.3, train=False, **rules)


# ---- inputs ----------------------------------------------------------------------------------------------


def _inputs(case, seed):
    """Name -> torch tensor on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TORCH[case["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    if case["kind"] == "xent":
        n, d, v = case["rows"], case["width"], case["vocab"]
        # rows as a final norm leaves them, weights whose logits spread by about 2
        got = dict(x=normal(n, d), w=normal(v, d, std=2.0 * d**-0.5), targets=whole(0, v, n))
        if case["ignored"]:
            got["targets"].masked_fill_(torch.rand(n, generator=g, device="cuda") < case["ignored"], -1)
        return got
    b, h, kv, t_q, t_k, dim = (case[n] for n in ("batch", "heads", "kv_heads", "t_q", "t_k", "dim"))
    # scores spread by 1; by 4 where they are capped, as the cap is there for large ones
    got = dict(q=normal(b, h, t_q, dim, std=4.0 if case["softcap"] else 1.0), k=normal(b, kv, t_k, dim), v=normal(b, kv, t_k, dim))
    if case["alibi"]:
        got["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
    if case["document"]:  # documents of that many tokens on average, one after another; some rows end in padding
        begins = torch.rand(b, t_k, generator=g, device="cuda") < 1.0 / case["document"]
        got["documents"] = begins.cumsum(1).to(torch.int32)
        pad = whole(0, 1 + t_k // 16, b, 1) * (torch.arange(b, device="cuda").reshape(b, 1) % 2)
        got["documents"].masked_fill_(torch.arange(t_k, device="cuda") >= t_k - pad, -1)
    if case["prefix"]:
        got["prefix"] = whole(0, 1 + t_k // 2, b)
    if case["ragged"]:  # a cache of t_k places, live to another length for each sequence
        got["lengths"] = whole(min(t_k, max(t_q, t_k // 4)), t_k + 1, b)
    if case["train"]:
        got["dout"] = normal(b, h, t_q, dim)
    return got


def prepare(case, seed):
    state = dict(case=dict(case), **_inputs(case, seed))
    if case["kind"] == "attend" and not case["train"]:  # a server's own buffers
        state["out"] = torch.empty_like(state["q"])
        state["lse"] = torch.empty(state["q"].shape[:-1], device="cuda")
    return state


# ---- the plain forms -------------------------------------------------------------------------------------


def _plain_rules(state):
    """(visible pairs, distances times slope or None) that broadcast with (b, kv, group, t_q, t_k)."""
    case = state["case"]
    b, t_q, t_k = case["batch"], case["t_q"], case["t_k"]
    key = torch.arange(t_k, device="cuda")
    length = state["lengths"].long() if case["ragged"] else torch.full((b,), t_k, device="cuda")
    at = length.reshape(b, 1) - t_q + torch.arange(t_q, device="cuda")  # (b, t_q)
    seen = (key < length.reshape(b, 1)).reshape(b, 1, t_k).expand(b, t_q, t_k)
    if case["causal"]:
        reach = key <= at.unsqueeze(-1)
        if case["prefix"]:
            reach = reach | (key < state["prefix"].reshape(b, 1, 1))
        seen = seen & reach
    if case["document"]:
        keys = state["documents"]
        rows = torch.gather(keys, 1, at.clamp(min=0))
        seen = seen & (rows.unsqueeze(-1) == keys.unsqueeze(1)) & (keys >= 0).unsqueeze(1)
    bias = None
    if case["alibi"]:
        far = (at.unsqueeze(-1) - key).abs().float()
        bias = state["slopes"].reshape(1, case["kv_heads"], -1, 1, 1) * far.reshape(b, 1, 1, t_q, t_k)
    return seen.reshape(b, 1, 1, t_q, t_k), bias


def _plain_attend(state):
    case = state["case"]
    b, h, kv, t_q, dim = (case[n] for n in ("batch", "heads", "kv_heads", "t_q", "dim"))
    scale, cap = dim**-0.5, case["softcap"]
    q = state["q"].float().reshape(b, kv, h // kv, t_q, dim)
    k, v = state["k"].float().unsqueeze(2), state["v"].float().unsqueeze(2)
    seen, bias = _plain_rules(state)
    flat = q.reshape(b, kv, -1, dim)  # a key head's query rows together
    s = (flat @ k.squeeze(2).transpose(-1, -2).contiguous()).reshape(b, kv, h // kv, t_q, -1).mul_(scale)
    bent = None
    if cap:
        bent = s.div_(cap).tanh_()
        s = bent * cap
    if bias is not None:
        s = s - bias
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf)
    p = p.div_(total.clamp(min=torch.finfo(torch.float32).tiny))
    out = (p.reshape(b, kv, -1, p.shape[-1]) @ v.squeeze(2)).reshape(b, kv, h // kv, t_q, dim)
    kind = state["q"].dtype
    if not case["train"]:
        return [out.reshape(b, h, t_q, dim).to(kind), lse.reshape(b, h, t_q)]
    do = state["dout"].float().reshape(b, kv, h // kv, t_q, dim)
    dp = (do.reshape(b, kv, -1, dim) @ v.squeeze(2).transpose(-1, -2).contiguous()).reshape(p.shape)
    ds = dp.sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    if cap:
        ds = ds.mul_(1 - bent * bent)
    ds = ds.mul_(scale).reshape(b, kv, -1, p.shape[-1])
    p = p.reshape(ds.shape)
    dq = ds @ k.squeeze(2)
    dk = ds.transpose(-1, -2).contiguous() @ flat
    dv = p.transpose(-1, -2).contiguous() @ do.reshape(b, kv, -1, dim)
    return [x.to(kind) for x in (out.reshape(b, h, t_q, dim), dq.reshape(b, h, t_q, dim), dk, dv)]


def _plain_xent(state):
    x, w, targets = state["x"].float(), state["w"].float(), state["targets"].long()
    live = targets >= 0
    at = targets.clamp(min=0).unsqueeze(1)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    p = (logits - top).exp_()
    total = p.sum(1, keepdim=True)
    count = live.sum().clamp(min=1)
    loss = torch.where(live, (top + total.log() - logits.gather(1, at)).squeeze(1), 0.0).sum() / count
    share = (live.float() / count).unsqueeze(1)
    dlogits = p.div_(total).scatter_add_(1, at, torch.full_like(share, -1.0)).mul_(share)
    return [loss, (dlogits @ w).to(state["x"].dtype), (dlogits.t() @ x).to(state["w"].dtype)]


# ---- the framework's calls -------------------------------------------------------------------------------

_programs = {}  # configuration -> its captured step, as a program holds one for its whole run


class _Held:
    """A torch tensor's memory as the bytes of a limn buffer."""

    __slots__ = ("ptr", "nbytes", "tensor")

    def __init__(self, tensor):
        self.ptr, self.nbytes, self.tensor = tensor.data_ptr(), tensor.numel() * tensor.element_size(), tensor


class _Bytes:
    """A limn device buffer as torch takes foreign memory; torch keeps this object, and so the buffer, alive."""

    __slots__ = ("buffer", "__cuda_array_interface__")

    def __init__(self, buffer, typestr, shape):
        self.buffer = buffer
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (buffer.ptr, False), "version": 2}


def _device():
    import limn_amd.hip  # noqa: F401  (registers "hip")
    from limn_amd.seam import active_device, set_device

    try:
        return active_device()
    except RuntimeError:
        set_device("hip")
        return active_device()


def _limn(x, trained):
    from limn_amd.seam import Node, Op, Tensor, bfloat16, float16, float32, int32

    dtype = {torch.float32: float32, torch.float16: float16, torch.bfloat16: bfloat16, torch.int32: int32}[x.dtype]
    t = Tensor.from_node(Node(Op.BUFFER, (), dtype, tuple(x.shape), _Held(x)))
    t.requires_grad = trained
    return t


def _torch(tensor):
    """A realized limn tensor's buffer as a torch tensor (no copy)."""
    name = tensor.dtype.name
    got = torch.as_tensor(_Bytes(tensor.node.arg, {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2"}[name], tensor.shape), device="cuda")
    return got.view(torch.bfloat16) if name == "bfloat16" else got


RULES = ("slopes", "documents", "prefix")


def _step(case):
    """The function that a program captures: limn tensors in, realized limn tensors out."""
    from limn_amd.seam import grad, realize

    if case["kind"] == "xent":
        from limn_amd.xent import linear_cross_entropy

        def head(x, w, targets):
            loss = linear_cross_entropy(x, w, targets)
            got = [loss, *grad(loss, [x, w])]
            realize(*got)
            return got

        return head
    from limn_amd.attend import attend

    names = [n for n, on in zip(RULES, (case["alibi"], case["document"], case["prefix"])) if on]

    def layer(q, k, v, dout, *rules):
        out = attend(q, k, v, causal=case["causal"], softcap=case["softcap"], **dict(zip(names, rules)))
        got = [out, *grad((out * dout).sum(), [q, k, v])]
        realize(*got)
        return got

    return layer


def _captured(state):
    _device()
    case = state["case"]
    names = ["x", "w", "targets"] if case["kind"] == "xent" else ["q", "k", "v", "dout", *(n for n in RULES if n in state)]
    args = [_limn(state[n], n in ("x", "w", "q", "k", "v")) for n in names]
    key = tuple(sorted((k, v) for k, v in case.items() if k != "name"))
    if key not in _programs:
        from limn_amd.seam import capture

        _programs[key] = capture(_step(case))
        for _ in range(2):  # the two calls that capture observes
            _programs[key](*args)
    return [_torch(t) for t in _programs[key](*args)]


def _served(state):
    """A server's call of the C ABI, on its own buffers and stream."""
    lib, case = _device().lib, state["case"]
    sizes = [case[n] for n in ("batch", "heads", "kv_heads", "t_q", "t_k", "dim", "dim")]
    if "workspace" not in state:
        need = lib.limn_hip_attend_workspace(CODE[case["dtype"]], *sizes, 0)
        state["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    at = [state[n].data_ptr() if n in state else None for n in ("q", "k", "v", *RULES, "lengths", "out", "lse")]
    status = lib.limn_hip_attend_fwd(*at, CODE[case["dtype"]], *sizes, int(case["causal"]), case["dim"] ** -0.5, case["softcap"],
                                     state["workspace"].data_ptr(), state["workspace"].numel(), torch.cuda.current_stream().cuda_stream)
    if status != 0:
        raise RuntimeError(f"limn_hip_attend_fwd: {lib.limn_hip_last_error().decode()}")
    return [state["out"], state["lse"]]


def run(state):
    if state["case"]["kind"] == "xent":
        return _captured(state) if own else _plain_xent(state)
    if own:
        return _captured(state) if state["case"]["train"] else _served(state)
    return _plain_attend(state)


# ---- the work no implementation can do without -----------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "xent":
        n, d, v = case["rows"], case["width"], case["vocab"]
        # x, w and the targets in, dx and dw out; the logits once (their second computing is a way of not keeping them) and two gradients
        return dict(bytes=2 * (n + v) * d * size + 4 * n, flops=6.0 * n * d * v)
    b, h, kv, t_q, t_k, dim = (case[n] for n in ("batch", "heads", "kv_heads", "t_q", "t_k", "dim"))
    live = 0.625 * t_k if case["ragged"] else float(t_k)  # lengths spread from a quarter of the cache to all of it
    if case["document"]:  # expected pairs of one row of tokens: a token's document began a geometric distance ago
        m = float(case["document"])
        before = sum(m * (1 - (1 - 1 / m) ** (i + 1)) for i in range(t_q))
        pairs = before if case["causal"] else 2 * before - t_q
        if case["prefix"]:
            pairs *= 1.125
    else:
        pairs = t_q * (live - (t_q - 1) / 2.0 if case["causal"] else live)
        if case["prefix"]:  # the upper triangle of a prefix of some quarter of the keys (its square's mean: a twelfth)
            pairs += t_q * t_q / 24.0 if t_q == t_k else 0
    q, k = b * h * t_q * dim * size, b * kv * live * dim * size
    unit = 2.0 * b * h * pairs * dim
    rules = 4 * h * case["alibi"] + 4 * b * t_k * bool(case["document"]) + 4 * b * case["prefix"] + 4 * b * case["ragged"]
    if case["train"]:  # q, k, v, dout in; out, dq, dk, dv out
        return dict(bytes=4 * q + 4 * k + rules, flops=7 * unit)
    return dict(bytes=2 * q + 2 * k + rules + 4 * b * h * t_q, flops=2 * unit)


# ---- the same values in 64 bits, from the definitions ----------------------------------------------------


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "xent":
        rows, w, targets = x["x"].double(), x["w"].double().requires_grad_(), x["targets"].long()
        if 3.0 * rows.numel() * case["vocab"] > 1.5e14:
            return None
        live = torch.nonzero(targets >= 0).squeeze(1)
        loss, dx, dw = torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros_like(rows), torch.zeros_like(w)
        for part in live.split(1024):  # some rows at a time: the logits are large
            r = rows[part].requires_grad_()
            here = torch.nn.functional.cross_entropy(r @ w.T, targets[part], reduction="sum") / len(live)
            dr, dpart = torch.autograd.grad(here, (r, w))
            loss, dw = loss + here.detach(), dw + dpart
            dx[part] = dr
        return [loss, dx, dw]
    b, h, kv, t_q, t_k, dim = (case[n] for n in ("batch", "heads", "kv_heads", "t_q", "t_k", "dim"))
    if b * h * float(t_q) * t_k * dim > 1e12:
        return None
    got = [torch.zeros(x[n].shape, dtype=torch.float64, device="cuda") for n in "qqkv"]
    lse = torch.empty(b, h, t_q, dtype=torch.float64, device="cuda")
    j = torch.arange(t_k, device="cuda")
    for n in range(b):
        length = int(x["lengths"][n]) if case["ragged"] else t_k
        i = torch.arange(length - t_q, length, device="cuda").unsqueeze(1)
        hide = (j >= length).expand(t_q, t_k)
        if case["causal"]:
            hide = hide | ((j > i) & (j >= (int(x["prefix"][n]) if case["prefix"] else 0)))
        if case["document"]:
            doc = x["documents"][n]
            own_doc = doc[i.clamp(min=0)]
            hide = hide | (own_doc != doc) | (own_doc < 0)
        empty = hide.all(1)
        for head in range(h):
            q, k, v = (x[m][n, head if m == "q" else head // (h // kv)].double().requires_grad_(case["train"]) for m in "qkv")
            s = torch.matmul(q, k.T) / math.sqrt(dim)
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            if case["alibi"]:
                s = s - x["slopes"][head].double() * (i - j).abs()
            s = s.masked_fill(hide, -math.inf)
            lse[n, head] = torch.logsumexp(s.detach(), 1)
            p = torch.softmax(s.masked_fill(empty.unsqueeze(1), 0.0), 1).masked_fill(empty.unsqueeze(1), 0.0)
            out = p @ v
            got[0][n, head] = out.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), x["dout"][n, head].double())
                got[1][n, head] = dq
                got[2][n, head // (h // kv)] += dk
                got[3][n, head // (h // kv)] += dv
    return got if case["train"] else [got[0], lse]
