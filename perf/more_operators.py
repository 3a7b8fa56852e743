"""The head's losses and the gated block with their gradients, as cases that can be timed.

A search over edits of a model scores rows of its final hidden states against
the vocabulary, and a program that looks for edits by gradients needs what
those scores and the feed-forward blocks below them hand back. The cases are
the operators of such a program:

  loss       the cross entropy of rows against a head over a large
             vocabulary: losses and log sums, no logits kept
  loss_grad  the same and its gradient: of the rows, and of the head where
             `dw` is set
  kl         the divergence of trial rows from base rows over the head's
             vocabulary (a trial's score), no logits kept
  kl_grad    the same and the gradient of the trial rows
  glu        act(x gate^T) * (x up^T) of rows
  glu_grad   its gradient: of the rows, and of both matrices where `dw` is set

Vocabularies and widths are those of the benchmark's configurations (a head of
128256 x 4096, 151936 x 896 and 151936 x 2048; blocks of 14336 x 4096 and
4864 x 896) and, in the drawn cases, any between small ones and these. Rows
are f32 (the model's own), bf16 or f16; weights bf16, f32, f16, or FP8 codes
with a scale for each 128 x 128 block, whose values are code * scale rounded
to bf16.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("silu", "gelu_tanh", "gelu", "relu", "relu2", "quick_gelu")  # by their numbers


# ---------------------------------------------------------------------------
# the cases

def _head(name, kind, dtype, fmt, n, vocab, hidden, dw=False):
    return dict(name=name, kind=kind, dtype=dtype, fmt=fmt, n=n, vocab=vocab, hidden=hidden, dw=dw)


def _glu(name, kind, dtype, fmt, n, inter, hidden, act="silu", dw=False):
    return dict(name=name, kind=kind, dtype=dtype, fmt=fmt, n=n, inter=inter, hidden=hidden, act=act, dw=dw)


def listed():
    return [
        # the loss of the next token of one prompt on the small model
        _head("loss_bf16_1", "loss", "bf16", "bf16", 1, 151936, 896),
        # the loss of every token of the headline batch: 64 prompts of 128 tokens
        _head("loss_bf16_8192", "loss", "bf16", "bf16", 8192, 128256, 4096),
        # one gradient for each of 64 prompts' last tokens, with respect to the model's own rows
        _head("loss_grad_f32_64", "loss_grad", "f32", "bf16", 64, 128256, 4096),
        # a training step of the small model's head, half-precision rows, a batch of no particular size
        _head("loss_grad_f16_1023", "loss_grad", "f16", "bf16", 1023, 151936, 896, dw=True),
        # a training step of a large head
        _head("loss_grad_bf16_4096", "loss_grad", "bf16", "bf16", 4096, 128256, 4096, dw=True),
        # a trial's score: 64 prompts' last tokens against the unedited model's
        _head("kl_f32_64", "kl", "f32", "bf16", 64, 128256, 4096),
        # edits sought by the gradient of the divergence over some answers' tokens
        _head("kl_grad_bf16_1500", "kl_grad", "bf16", "bf16", 1500, 151936, 2048),
        # the small model's block on a single token
        _glu("glu_bf16_1", "glu", "bf16", "bf16", 1, 4864, 896),
        # a few short prompts on 8-bit weights, the model's own rows
        _glu("glu_f32_fp8_100", "glu", "f32", "fp8", 100, 14336, 4096),
        # the headline batch
        _glu("glu_bf16_8192", "glu", "bf16", "bf16", 8192, 14336, 4096),
        # the small model's block in f32, rows and weights
        _glu("glu_grad_f32_300", "glu_grad", "f32", "f32", 300, 4864, 896, dw=True),
        # a training step of a large block
        _glu("glu_grad_bf16_4096", "glu_grad", "bf16", "bf16", 4096, 14336, 4096, dw=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    kind = rng.choice(["loss", "loss_grad", "kl", "kl_grad", "glu", "glu_grad"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    fmt = rng.choice(["bf16", "bf16", "bf16", "f32", "f16", "fp8"])
    hidden = rng.choice([896, 2048, 4096, _log(rng, 40, 4096)])
    dw = kind.endswith("_grad") and kind != "kl_grad" and rng.random() < 0.5
    exact_rows = dtype == "f32" or fmt in ("f32", "f16")
    n = _log(rng, 1, 8192)
    if kind.startswith("glu"):
        inter = rng.choice([4864, 14336, _log(rng, 100, 14336)])
        while n * inter * hidden > (6e10 if exact_rows else 2.4e11):
            n = max(1, n // 2)
        act = rng.choice(["silu", "silu", "gelu_tanh", "gelu", "quick_gelu"])
        return _unnamed(_glu("", kind, dtype, fmt, n, inter, hidden, act, dw))
    vocab = rng.choice([128256, 151936, _log(rng, 1000, 151936)])
    while n * vocab * hidden > (5e11 if exact_rows else 2e12):
        n = max(1, n // 2)
    return _unnamed(_head("", kind, dtype, fmt, n, vocab, hidden, dw))


def _rows_of(case):
    return case["vocab"] if "vocab" in case else case["inter"]


def work(case):
    e = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    n, h, r = case["n"], case["hidden"], _rows_of(case)
    wb = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "fp8": 1 + 4 / 16384}[case["fmt"]] * r * h
    x, product, kind, dw = n * h * e, 2.0 * n * r * h, case["kind"], case["dw"]
    if kind == "loss":
        return {"bytes": x + wb + 12 * n, "flops": product}
    if kind == "loss_grad":
        return {"bytes": 2 * x + wb + 16 * n + dw * r * h * e, "flops": (2 + dw) * product}
    if kind == "kl":
        return {"bytes": 2 * x + wb + 12 * n, "flops": 2 * product}
    if kind == "kl_grad":
        return {"bytes": 3 * x + wb + 16 * n, "flops": 3 * product}
    if kind == "glu":
        return {"bytes": x + 2 * wb + n * r * e, "flops": 2 * product}
    return {"bytes": 2 * x + 2 * wb + n * r * e + 2 * dw * r * h * e, "flops": (4 + 2 * dw) * product}


# ---------------------------------------------------------------------------
# inputs

class _State:
    """What a user's program holds."""

    tensors = ()

    def __del__(self):
        for t in self.tensors:
            t.free()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _weight(fmt, rows, cols, gen):
    """A weight as it is stored: a tensor, or (codes, scales of 128 x 128 blocks)."""
    w = torch.randn(rows, cols, generator=gen, device="cuda") * 0.02
    if fmt != "fp8":
        return w.to(DTYPES[fmt])
    sr, sc = -(-rows // 128), -(-cols // 128)
    w = torch.nn.functional.pad(w, (0, sc * 128 - cols, 0, sr * 128 - rows)).view(sr, 128, sc, 128)
    scale = (w.abs().amax((1, 3)).clamp_min(1e-12) / 448).float()
    codes = (w / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(sr * 128, sc * 128)
    return codes[:rows, :cols].contiguous(), scale


def _decoded(w):
    """The values of a stored weight in 32 bits."""
    if not isinstance(w, tuple):
        return w.float()
    codes, scale = w
    scale = scale.repeat_interleave(128, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]
    return (codes.view(torch.float8_e4m3fn).float() * scale).to(torch.bfloat16).float()


def prepare(case, seed):
    s = _State()
    s.case, s.calls = case, None
    gen, t = _gen(seed), DTYPES[case["dtype"]]
    n, h, r = case["n"], case["hidden"], _rows_of(case)
    x = torch.randn(n, h, generator=gen, device="cuda")
    if "vocab" not in case:
        s.x = x.to(t)
        s.w = [_weight(case["fmt"], r, h, gen) for _ in range(2)]
        if case["kind"] == "glu_grad":
            s.dout = (torch.randn(n, r, generator=gen, device="cuda") * 0.1).to(t)
    else:
        s.w = [_weight(case["fmt"], r, h, gen)]
        s.targets = torch.randint(0, r, (n,), generator=gen, device="cuda", dtype=torch.int32)
        # every other token is one that the model is rather sure of
        rows = _decoded(s.w[0])[s.targets.long()]
        sure = torch.rand(n, 1, generator=gen, device="cuda") * 10 * (torch.arange(n, device="cuda") % 2)[:, None]
        x += rows * (sure / rows.square().sum(1, keepdim=True))
        del rows
        # a tenth of the rows has no target
        s.targets[torch.rand(n, generator=gen, device="cuda") < 0.1] = -100
        s.x = x.to(t)
        if case["kind"].startswith("kl"):
            s.trial = (x + 0.5 * torch.randn(n, h, generator=gen, device="cuda")).to(t)
        # the weights of a mean; half precision scales its loss
        s.dloss = (0.5 + torch.rand(n, generator=gen, device="cuda")) * ((4096 if case["dtype"] == "f16" else 1) / n)
    if own:  # the registered weights that a user's program keeps beside its rows
        s.tensors = [_upload(w, case["fmt"]) for w in s.w]
        torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the plain form

def _log_sum(logits):
    top = logits.amax(-1, keepdim=True)
    return (logits - top).exp_().sum(-1).log_() + top[:, 0]


def _plain_loss(s):
    w, x = _decoded(s.w[0]), s.x.float()
    logits = torch.matmul(x, w.T)
    lse = _log_sum(logits)
    target = s.targets.long()
    live, at = target >= 0, target.clamp(min=0)[:, None]
    loss = torch.where(live, lse - logits.gather(1, at)[:, 0], 0)
    if s.case["kind"] == "loss":
        return {"loss": loss, "lse": lse}
    d = logits.sub_(lse[:, None]).exp_()
    d.scatter_add_(1, at, torch.full_like(lse, -1)[:, None])
    d.mul_(torch.where(live, s.dloss, 0)[:, None])
    out = {"loss": loss, "lse": lse, "dx": torch.matmul(d, w).to(s.x.dtype)}
    if s.case["dw"]:
        out["dw"] = torch.matmul(d.T, x).to(s.x.dtype)
    return out


def _plain_kl(s):
    w = _decoded(s.w[0])
    # where f32 gradients are wanted the logits in 64 bits: in the difference of p and q, which are near each other,
    # 32 lose what the gradients hold
    t = torch.float64 if s.case["kind"] == "kl_grad" and s.case["dtype"] == "f32" else torch.float32
    p, q = (torch.matmul(x.to(t), w.to(t).T).double() for x in (s.x, s.trial))
    lse_p, lse_q = _log_sum(p), _log_sum(q)
    p, q = p.sub_(lse_p[:, None]), q.sub_(lse_q[:, None])
    kl = (p.exp() * (p - q)).sum(-1)
    out = {"kl": kl.float(), "lse_base": lse_p.float(), "lse_trial": lse_q.float()}
    if s.case["kind"] == "kl_grad":
        d = q.exp_().sub_(p.exp_()).float().mul_(s.dloss[:, None])
        out["dx"] = torch.matmul(d, w).to(s.x.dtype)
    return out


def _act(a, g):
    """The activation of g and its derivative."""
    if a == "silu":
        t = 1 / (1 + (-g).exp())
        return g * t, t * (1 + g * (1 - t))
    if a == "quick_gelu":
        t = 1 / (1 + (-1.702 * g).exp())
        return g * t, t * (1 + 1.702 * g * (1 - t))
    if a == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * (-0.5 * g * g).exp() * (1 / math.sqrt(2 * math.pi))
    if a == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    r = g.clamp(min=0)
    return (r, (g > 0).to(g.dtype)) if a == "relu" else (r * r, 2 * r)


def _plain_glu(s):
    x, (wg, wu) = s.x.float(), (_decoded(w) for w in s.w)
    u = torch.matmul(x, wu.T)
    y, dy = _act(s.case["act"], torch.matmul(x, wg.T))
    if s.case["kind"] == "glu":
        return (y * u).to(s.x.dtype)
    d = s.dout.float()
    dg, du = d * u * dy, d * y
    out = {"dx": (torch.matmul(dg, wg) + torch.matmul(du, wu)).to(s.x.dtype)}
    if s.case["dw"]:
        out["dgate"] = torch.matmul(dg.T, x).to(s.x.dtype)
        out["dup"] = torch.matmul(du.T, x).to(s.x.dtype)
    return out


# ---------------------------------------------------------------------------
# the framework's operators

_dev = None


def _device():
    global _dev
    if _dev is None:
        from ditch_amd.hip import Device
        _dev = Device(0)
    return _dev


def _upload(w, fmt):
    from ditch_amd.weights import HostWeight
    if fmt == "fp8":
        return _device().upload(HostWeight.fp8(w[0].cpu().numpy(), w[1].cpu().numpy(), 128, 128))
    if fmt == "bf16":
        return _device().upload(HostWeight.bf16(w.view(torch.int16).cpu().numpy().view("uint16")))
    return _device().upload((HostWeight.f32 if fmt == "f32" else HostWeight.f16)(w.cpu().numpy()))


def _calls(s):
    """The buffers and their descriptors that a user's program makes once."""
    case, dev, t = s.case, _device(), DTYPES[s.case["dtype"]]
    n, c = case["n"], _State()

    def rows(x):
        return dev.kv_rows(x.data_ptr(), x.numel() * x.element_size(), x.shape[1])

    def rows_like(r, cols):
        x = torch.empty(r, cols, dtype=t, device="cuda")
        return x, rows(x)

    c.x, w = rows(s.x), s.tensors[0]
    kind, dtype, dw = case["kind"], case["dtype"], case["dw"]
    if kind == "glu":
        c.out, c.out_rows = rows_like(n, case["inter"])
        c.bytes = w.glu_rows_workspace(s.tensors[1], n, dtype)
    elif kind == "glu_grad":
        c.dout = rows(s.dout)
        c.bytes = w.glu_rows_grad_workspace(s.tensors[1], n, dtype, dw=dw)
        c.dw = [rows_like(case["inter"], case["hidden"]) if dw else (None, None) for _ in range(2)]
    else:
        c.one, c.lse, c.lse_trial = (torch.empty(n, device="cuda") for _ in range(3))
        if kind.startswith("kl"):
            c.trial = rows(s.trial)
            c.bytes = w.head_kl_workspace(n, dtype)
            if kind == "kl_grad":
                c.bytes = max(c.bytes, w.head_kl_grad_workspace(n, dtype))
        else:
            c.bytes = w.head_loss_workspace(n, dtype)
            if kind == "loss_grad":
                c.bytes = max(c.bytes, w.head_loss_grad_workspace(n, dtype, dw=dw))
            c.dw = [rows_like(case["vocab"], case["hidden"]) if dw else (None, None)]
    if kind.endswith("_grad"):
        c.dx, c.dx_rows = rows_like(n, case["hidden"])
    c.ws = torch.empty(max(c.bytes, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return c


def _own(s):
    case = s.case
    if s.calls is None:
        s.calls = _calls(s)
    c, kind, dtype, n, w = s.calls, case["kind"], case["dtype"], case["n"], s.tensors[0]
    ws = (c.ws.data_ptr(), c.bytes)
    if kind == "glu":
        w.glu_rows(s.tensors[1], dtype, c.out_rows, c.x, n, *ws, act=ACTS.index(case["act"]))
        return c.out
    if kind == "glu_grad":
        w.glu_rows_grad(s.tensors[1], dtype, c.dx_rows, c.dw[0][1], c.dw[1][1], c.dout, c.x, n, *ws,
                        act=ACTS.index(case["act"]))
        return {"dx": c.dx, "dgate": c.dw[0][0], "dup": c.dw[1][0]} if case["dw"] else {"dx": c.dx}
    if kind.startswith("kl"):
        w.head_kl(dtype, c.one.data_ptr(), c.lse.data_ptr(), c.lse_trial.data_ptr(), c.x, c.trial, n, *ws)
        out = {"kl": c.one, "lse_base": c.lse, "lse_trial": c.lse_trial}
        if kind == "kl_grad":
            w.head_kl_grad(dtype, c.dx_rows, c.x, c.trial, n, c.lse.data_ptr(), c.lse_trial.data_ptr(),
                           s.dloss.data_ptr(), *ws)
            out["dx"] = c.dx
        return out
    w.head_loss(dtype, c.one.data_ptr(), c.lse.data_ptr(), c.x, n, s.targets.data_ptr(), *ws)
    out = {"loss": c.one, "lse": c.lse}
    if kind == "loss_grad":
        w.head_loss_grad(dtype, c.dx_rows, c.dw[0][1], c.x, n, s.targets.data_ptr(), c.lse.data_ptr(),
                         s.dloss.data_ptr(), *ws)
        out["dx"] = c.dx
        if case["dw"]:
            out["dw"] = c.dw[0][0]
    return out


def run(s):
    if own:
        return _own(s)
    kind = s.case["kind"]
    return _plain_glu(s) if kind.startswith("glu") else _plain_kl(s) if kind.startswith("kl") else _plain_loss(s)


# ---------------------------------------------------------------------------
# the definition in 64 bits

BLOCK = 1024  # rows at a time


def _values64(w):
    """The values of a stored weight: an FP8 block's codes times its scale as bf16, else the numbers themselves."""
    if not isinstance(w, tuple):
        return w.double()
    codes, scale = w
    out = torch.empty(codes.shape, dtype=torch.float64, device="cuda")
    for i in range(scale.shape[0]):
        block = codes[i * 128:(i + 1) * 128].view(torch.float8_e4m3fn).float()
        each = scale[i].repeat_interleave(128)[:codes.shape[1]]
        out[i * 128:(i + 1) * 128] = (block * each).bfloat16().double()
    return out


def _exact_loss(case, s):
    w = _values64(s.w[0])
    loss, lse, dx = [], [], []
    dw = torch.zeros_like(w) if case["dw"] else None
    for i in range(0, case["n"], BLOCK):
        x, t = s.x[i:i + BLOCK].double(), s.targets[i:i + BLOCK].long()
        some = (t >= 0).double()
        logits = x @ w.T
        lse.append(torch.logsumexp(logits, 1))
        picked = (x * w[t.clamp(min=0)]).sum(1)
        loss.append((lse[-1] - picked) * some)
        if case["kind"] == "loss_grad":
            weight = s.dloss[i:i + BLOCK].double() * some
            p = logits.softmax(1) * weight[:, None]
            dx.append(p @ w - weight[:, None] * w[t.clamp(min=0)])
            if dw is not None:
                dw += p.T @ x
                dw.index_add_(0, t.clamp(min=0), -weight[:, None] * x)
    out = {"loss": torch.cat(loss), "lse": torch.cat(lse)}
    if dx:
        out["dx"] = torch.cat(dx)
    if dw is not None:
        out["dw"] = dw
    return out


def _exact_kl(case, s):
    w = _values64(s.w[0])
    got = {"kl": [], "lse_base": [], "lse_trial": []} | ({"dx": []} if case["kind"] == "kl_grad" else {})
    for i in range(0, case["n"], BLOCK):
        p, q = s.x[i:i + BLOCK].double() @ w.T, s.trial[i:i + BLOCK].double() @ w.T
        got["lse_base"].append(p.logsumexp(1))
        got["lse_trial"].append(q.logsumexp(1))
        p, q = p.log_softmax(1), q.log_softmax(1)
        got["kl"].append(torch.nn.functional.kl_div(q, p, reduction="none", log_target=True).sum(1))
        if "dx" in got:
            got["dx"].append(((q.exp() - p.exp()) * s.dloss[i:i + BLOCK].double()[:, None]) @ w)
    return {k: torch.cat(v) for k, v in got.items()}


def _exact_glu(case, s):
    wg, wu = (_values64(w) for w in s.w)
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh"), "relu": torch.relu,
         "relu2": lambda g: torch.relu(g) ** 2, "quick_gelu": lambda g: g * torch.sigmoid(1.702 * g)}[case["act"]]
    rows, dwg, dwu = [], torch.zeros_like(wg), torch.zeros_like(wu)
    for i in range(0, case["n"], BLOCK):
        x = s.x[i:i + BLOCK].double()
        g, u = (x @ wg.T).requires_grad_(), (x @ wu.T).requires_grad_()
        y = f(g) * u
        if case["kind"] == "glu":
            rows.append(y.detach())
            continue
        dg, du = torch.autograd.grad(y, (g, u), s.dout[i:i + BLOCK].double())
        rows.append(dg @ wg + du @ wu)
        if case["dw"]:
            dwg += dg.T @ x
            dwu += du.T @ x
    if case["kind"] == "glu":
        return torch.cat(rows)
    return {"dx": torch.cat(rows)} | ({"dgate": dwg, "dup": dwu} if case["dw"] else {})


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return (_exact_glu if kind.startswith("glu") else _exact_kl if kind.startswith("kl") else _exact_loss)(case, s)
