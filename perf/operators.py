"""The paged 8-bit cache and the beam step, as cases that can be timed.

Generation over long contexts keeps its keys and values in pages of 8-bit
codes, with one scale for each page and head. The cases are the operators
that such a program calls between the model's products:

  append   new keys and values, rotated to their positions, quantised into
           the cache's pages, and the queries rotated with them; then the
           touched pages read back as rows (what a step writes and what an
           export or a prefix hand-over reads)
  attn     attention of new rows over the cached sequences: decode steps (a
           row a sequence), chunks of prompts, full causal or a sliding window
           with the first tokens kept visible
  beam     the best continuations over beams and vocabulary
  fork     the beams' states reordered by the chosen parents: page tables and
           the contents of partly filled pages, in every layer

Head shapes and vocabularies are those of the benchmark's configurations
(32/8 heads of 128, 14/2 heads of 64, 32/4 heads of 128, latent attention's
192/128) and some generic ones.

The page format (both sides read and write it): codes [layers][pages]
[kv_heads][page bytes], a head's keys in front of its values. Keys: per 16
tokens and 64 dims [4][16 tokens][16 dims]. Values: per 32 tokens and 32 dims
[4 g][16 dims d][2 h][8 j], dim 16 h + d, token 16 (j / 4) + 4 g + j % 4. Head
dims pad to multiples of 64 with zeros. Scales [layers][pages][kv_heads][2].
"""
import math

import torch

own = False

MOST_CODE = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# the cases

def _append(name, cache, dtype, heads, kv_heads, head_dim, v_head_dim, page, seqs, rows, pos, ragged, rotary, style):
    return dict(name=name, kind="append", cache=cache, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                v_head_dim=v_head_dim, page=page, seqs=seqs, rows=rows, pos=pos, ragged=ragged, rotary=rotary,
                style=style)


def _attn(name, cache, dtype, heads, kv_heads, head_dim, v_head_dim, page, seqs, rows, pos, ragged, window, sinks):
    return dict(name=name, kind="attn", cache=cache, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                v_head_dim=v_head_dim, page=page, seqs=seqs, rows=rows, pos=pos, ragged=ragged, window=window,
                sinks=sinks)


def _beam(name, prompts, beams, vocab, k):
    return dict(name=name, kind="beam", prompts=prompts, beams=beams, vocab=vocab, k=k)


def _fork(name, cache, layers, kv_heads, head_dim, page, prompts, beams, length):
    return dict(name=name, kind="fork", cache=cache, layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page,
                prompts=prompts, beams=beams, length=length)


def listed():
    return [
        # a decode step of 64 sequences somewhere inside their pages
        _append("append_int8_64x1", "int8", "bf16", 32, 8, 128, 128, 64, 64, 1, 1000, True, 128, "neox"),
        # a batch of prompts of different lengths, f32 activations, on top of cached prefixes
        _append("append_e4m3_24x500", "e4m3", "f32", 32, 8, 128, 128, 64, 24, 500, 130, True, 128, "neox"),
        # one prompt's decode step: latency
        _attn("decode_int8_1x500", "int8", "f32", 32, 8, 128, 128, 64, 1, 1, 499, False, 0, 0),
        # a full decode batch over long contexts of different lengths
        _attn("decode_int8_64x8192", "int8", "bf16", 32, 8, 128, 128, 64, 64, 1, 8191, True, 0, 0),
        # one very long context: the keys split over the chip
        _attn("decode_e4m3_1x130001", "e4m3", "f32", 32, 4, 128, 128, 128, 1, 1, 130000, False, 0, 0),
        # long chats decoded with a window and the first tokens visible
        _attn("decode_window_48x20000", "int8", "f32", 14, 2, 64, 64, 64, 48, 1, 20000, True, 1024, 4),
        # a chunk of two prompts on top of what is cached
        _attn("chunk_e4m3_2x2048", "e4m3", "bf16", 32, 8, 128, 128, 64, 2, 2048, 2048, False, 0, 0),
        # ragged prompts under the window, f32 activations
        _attn("chunk_window_5x1500", "int8", "f32", 14, 2, 64, 64, 32, 5, 1500, 700, True, 512, 8),
        # the beam step of one prompt, and of a full batch
        _beam("beam_1x4", 1, 4, 151936, 8),
        _beam("beam_64x8", 64, 8, 128256, 16),
        # their states: the small model's, and a 32-layer one's
        _fork("fork_1x4", "int8", 24, 2, 64, 64, 1, 4, 100),
        _fork("fork_16x8", "e4m3", 32, 8, 128, 64, 16, 8, 750),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "attn", "beam", "fork"])
    cache = rng.choice(["int8", "e4m3"])
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        vocab = _log(rng, 500, 152000)
        prompts = _log(rng, 1, max(1, min(100, 64 * 8 * 128256 // (beams * vocab))))
        return {k: v for k, v in _beam("", prompts, beams, vocab, rng.choice([beams, 2 * beams])).items()
                if k != "name"}
    if kind == "fork":
        layers, kv_heads, head_dim = rng.randint(1, 32), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128])
        prompts, beams = _log(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8])
        case = _fork("", cache, layers, kv_heads, head_dim, rng.choice([32, 64]), prompts, beams, _log(rng, 1, 800))
        return {k: v for k, v in case.items() if k != "name"}
    dtype = rng.choice(["f32", "bf16", "f16"])
    kv_heads, (hd, vd) = rng.choice([1, 2, 3, 4, 8]), rng.choice([(64, 64), (128, 128), (128, 128), (80, 80),
                                                                  (192, 128), (256, 256)])
    heads, page = kv_heads * rng.choice([1, 2, 4, 7, 8]), rng.choice([32, 64, 128])
    if kind == "append":
        rows = _log(rng, 1, 700)
        each = (rows + page) * kv_heads * (hd + vd) * 9 + rows * heads * hd * 8  # bytes of a sequence, about
        case = _append("", cache, dtype, heads, kv_heads, hd, vd, page, _log(rng, 1, max(1, 390_000_000 // each)), rows,
                       rng.randint(0, 2000), rng.random() < 0.7, rng.choice([hd, hd // 2]),
                       rng.choice(["neox", "gptj"]))
    else:
        wide = rng.random() < 0.5
        window, sinks = (0, 0) if wide else (_log(rng, 1, 2000), rng.choice([0, 1, 4, 33]))
        if rng.random() < 0.55:
            rows = rng.choice([1, 1, 1, 2, 5])
            pos = _log(rng, 1, 60000)
            seqs = _log(rng, 1, max(1, min(64, 500_000_000 // (pos * kv_heads * (hd + vd)))))
        else:
            rows = _log(rng, 8, 1500)
            pos = rng.choice([0, _log(rng, 1, 3000)])
            # (the plain form holds every head's scores)
            most = 400_000_000 * 256 // (hd + vd) // heads
            rows = min(rows, max(8, most // (rows + pos)))
            seqs = _log(rng, 1, max(1, min(8, most // (rows * (rows + pos)))))
        case = _attn("", cache, dtype, heads, kv_heads, hd, vd, page, seqs, rows, pos, rng.random() < 0.7, window,
                     sinks)
    return {k: v for k, v in case.items() if k != "name"}


def _rows_pos(case):
    """Each sequence's new rows and the position of the first: the case's, or,
    ragged, up to them (in a larger batch some sequences have none)."""
    rows, pos = [case["rows"]], [case["pos"]]
    for b in range(1, case["seqs"]):
        r, p = case["rows"], case["pos"]
        if case["ragged"]:
            r = 0 if b % 9 == 8 else r - b * 7919 % (r - r // 3) if r > 1 else 1
            p = p - b * 104729 % (p // 2 + 1)
        rows.append(r)
        pos.append(p)
    return rows, pos


def _padded(dim):
    return -(-dim // 64) * 64


def work(case):
    if case["kind"] == "beam":
        n = case["prompts"] * case["beams"]
        return {"bytes": 4.0 * n * (case["vocab"] + 1) + 12.0 * case["prompts"] * case["k"],
                "flops": 4.0 * n * case["vocab"]}
    if case["kind"] == "fork":
        # the tables in and out; a copy for each child whose parent an earlier one took over (on average 1/e of them)
        n, cols = case["prompts"] * case["beams"], -(-case["length"] // case["page"]) + 1
        used = case["length"] % case["page"]
        moved = n * (1 - 1 / case["beams"]) ** case["beams"] if used else 0
        token = case["layers"] * case["kv_heads"] * 2 * case["head_dim"]
        return {"bytes": 2.0 * moved * (token * used + 8 * case["layers"] * case["kv_heads"]) + 8.0 * n * (cols + 2),
                "flops": 0}
    rows, pos = _rows_pos(case)
    e = 4 if case["dtype"] == "f32" else 2
    width = case["kv_heads"] * (case["head_dim"] + case["v_head_dim"])
    if case["kind"] == "append":
        # rows in (keys, values, queries), codes out and in again, rows out
        read = sum(r + p % case["page"] if r else 0 for r, p in zip(rows, pos))
        n = sum(rows)
        return {"bytes": float(n * width * (e + 1) + read * width * 5 + 2 * n * case["heads"] * case["head_dim"] * e),
                "flops": 6.0 * n * width}
    pairs, keys = 0, 0
    for r, p in zip(rows, pos):
        w, s = case["window"], case["sinks"]
        if r == 0:
            continue
        if not w:
            pairs += r * p + r * (r + 1) // 2
            keys += r + p
        else:
            first = max(0, p - w + 1)
            keys += r + p - first + min(s, first)
            for t in range(p, p + r):
                lo = max(0, t - w + 1)
                pairs += t - lo + 1 + min(s, lo)
    out = sum(rows) * case["heads"] * (case["head_dim"] + case["v_head_dim"]) * e
    return {"bytes": float(keys * width + out), "flops": 2.0 * pairs * case["heads"] * (case["head_dim"] +
                                                                                         case["v_head_dim"])}


# ---------------------------------------------------------------------------
# inputs

class _State:
    """What a user's program holds."""


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(rows):
    at = [0]
    for r in rows:
        at.append(at[-1] + r)
    return at


def _pool(s, case, layers, n_pages, gen):
    """A cache whose pages hold normal keys and values of about unit size, some
    channels of the keys larger than others."""
    dk, dv = _padded(case["head_dim"]), _padded(case.get("v_head_dim", case["head_dim"]))
    kvh, page = case["kv_heads"], case["page"]
    shape = (layers, n_pages, kvh, page // 16)
    channel = 0.5 + torch.rand(dk // 64, 4, 1, 16, generator=gen, device="cuda") * 1.5
    channel.view(-1)[::37] *= 3
    spread = {"int8": 28.0, "e4m3": 90.0}[case["cache"]]
    k = torch.randn(*shape, dk // 64, 4, 16, 16, generator=gen, device="cuda") * (channel / channel.max() * 1.5)
    v = torch.randn(layers, n_pages, kvh, page // 32, dv // 32, 4, 16, 2, 8, generator=gen, device="cuda")
    # the dims a head does not have are zero
    dims = torch.arange(dk, device="cuda").view(dk // 64, 4, 1, 16)
    k *= dims < case["head_dim"]
    dims = torch.arange(dv, device="cuda").view(dv // 32, 1, 2, 16).permute(0, 1, 3, 2).unsqueeze(-1)
    v *= dims < case.get("v_head_dim", case["head_dim"])
    parts = [x.reshape(layers, n_pages, kvh, -1).mul_(spread) for x in (k, v)]
    del k, v
    s.codes = torch.empty(layers, n_pages, kvh, page * (dk + dv), dtype=torch.uint8, device="cuda")
    at = 0
    for x in parts:
        x.clamp_(-MOST_CODE[case["cache"]], MOST_CODE[case["cache"]])
        code = x.round_().to(torch.int8) if case["cache"] == "int8" else x.to(torch.float8_e4m3fn)
        s.codes[..., at:at + x.shape[-1]] = code.view(torch.uint8)
        at += x.shape[-1]
    s.scales = (0.8 + 0.4 * torch.rand(layers, n_pages, kvh, 2, generator=gen, device="cuda")) / spread


def _sequences(s, case, gen):
    rows, pos = _rows_pos(case)
    pages = [-(-(r + p) // case["page"]) for r, p in zip(rows, pos)]
    s.n_rows, s.max_rows, s.max_len = sum(rows), max(rows), max(r + p for r, p in zip(rows, pos))
    s.cols = max(max(pages), 1)
    n_pages = sum(pages) + 3
    _pool(s, case, 1, n_pages, gen)
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    s.table = torch.full((case["seqs"], s.cols), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        s.table[b, :n] = ids[at:at + n]
        at += n
    s.starts, s.pos = _i32(_starts(rows)), _i32(pos)


def prepare(case, seed):
    s = _State()
    s.case, s.calls = case, None
    gen = _gen(seed)
    if case["kind"] == "beam":
        n = case["prompts"] * case["beams"]
        s.logits = torch.randn(n, case["vocab"], generator=gen, device="cuda") * 2.5
        s.prev = -torch.rand(case["prompts"], case["beams"], generator=gen, device="cuda") * 6
        s.scores = torch.zeros(case["prompts"], case["k"], device="cuda")
        s.parents = torch.zeros(case["prompts"], case["k"], dtype=torch.int32, device="cuda")
        s.tokens = torch.zeros(case["prompts"], case["k"], dtype=torch.int32, device="cuda")
        return s
    if case["kind"] == "fork":
        n, used = case["prompts"] * case["beams"], -(-case["length"] // case["page"])
        s.cols = used + 1
        # the full pages are shared by a prompt's beams; the last one is each beam's own, and so is its spare
        own_pages, shared = 3 * n, case["prompts"] * (used - 1)
        _pool(s, case, case["layers"], own_pages + shared, gen)
        ids = torch.randperm(own_pages + shared, generator=gen, device="cuda").to(torch.int32)
        s.table = torch.empty(case["prompts"], case["beams"], s.cols, dtype=torch.int32, device="cuda")
        s.table[:, :, used - 1:] = ids[:2 * n].view(case["prompts"], case["beams"], 2)
        s.table[:, :, :used - 1] = ids[3 * n:].view(case["prompts"], 1, used - 1)
        s.table = s.table.view(n, s.cols)
        s.spare = ids[2 * n:3 * n].clone()
        s.parents = torch.randint(0, case["beams"], (n,), generator=gen, device="cuda", dtype=torch.int32)
        s.lens = torch.full((case["prompts"],), case["length"], dtype=torch.int32, device="cuda")
        s.table_out, s.spare_out = torch.zeros_like(s.table), torch.zeros_like(s.spare)
        return s
    _sequences(s, case, gen)
    t, kvh, hd, vd = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"], case["v_head_dim"]
    s.q = (torch.randn(s.n_rows, case["heads"], hd, generator=gen, device="cuda") * 1.5).to(t)
    if case["kind"] == "attn":
        s.out = torch.zeros(s.n_rows, case["heads"], vd, dtype=t, device="cuda")
        return s
    s.k = torch.randn(s.n_rows, kvh, hd, generator=gen, device="cuda").to(t)
    s.v = torch.randn(s.n_rows, kvh, vd, generator=gen, device="cuda").to(t)
    half = case["rotary"] // 2
    angle = torch.arange(s.max_len, dtype=torch.float64, device="cuda")[:, None] * \
        5e5 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    s.cos, s.sin = angle.cos().float(), angle.sin().float()
    # what is read back: from the start of the page of each sequence's first new row
    rows, pos = _rows_pos(case)
    back = [r + p % case["page"] if r else 0 for r, p in zip(rows, pos)]
    s.n_back, s.max_back = sum(back), max(back)
    s.back_starts = _i32(_starts(back))
    s.back_pos = _i32([p - p % case["page"] for p in pos])
    s.q_out = torch.zeros_like(s.q)
    s.k_out = torch.zeros(s.n_back, kvh, hd, device="cuda")
    s.v_out = torch.zeros(s.n_back, kvh, vd, device="cuda")
    return s


# ---------------------------------------------------------------------------
# the plain form

def _values(codes, cache):
    return (codes.view(torch.int8) if cache == "int8" else codes.view(torch.float8_e4m3fn)).float()


def _unpack(codes, case):
    """Keys [..., page, dk] and values [..., page, dv] (codes' values) of pages of codes [..., page bytes]."""
    dk, dv = _padded(case["head_dim"]), _padded(case.get("v_head_dim", case["head_dim"]))
    page, lead = case["page"], codes.shape[:-1]
    x = _values(codes, case["cache"])
    k = x[..., :page * dk].reshape(-1, page // 16, dk // 64, 4, 16, 16).permute(0, 1, 4, 2, 3, 5)
    v = x[..., page * dk:].reshape(-1, page // 32, dv // 32, 4, 16, 2, 2, 4).permute(0, 1, 6, 3, 7, 2, 5, 4)
    return k.reshape(*lead, page, dk), v.reshape(*lead, page, dv)


def _pack(k, v, case):
    """_unpack's inverse: codes from code values."""
    t = torch.int8 if case["cache"] == "int8" else torch.float8_e4m3fn
    lead, page, dk, dv = k.shape[:-2], k.shape[-2], k.shape[-1], v.shape[-1]
    k = k.reshape(-1, page // 16, 16, dk // 64, 4, 16).permute(0, 1, 3, 4, 2, 5).reshape(-1, page * dk)
    v = v.reshape(-1, page // 32, 2, 4, 4, dv // 32, 2, 16).permute(0, 1, 5, 3, 7, 6, 2, 4).reshape(-1, page * dv)
    return torch.cat((k, v), -1).float().to(t).view(torch.uint8).reshape(*lead, -1)


def _round(y, cache):
    """The nearest code values of y (64 bits, ties to even)."""
    most = MOST_CODE[cache]
    y = y.clamp(-most, most)
    if cache == "int8":
        return y.round()
    step = torch.exp2((torch.frexp(y).exponent - 1).clamp(min=-6).double() - 3)
    return (y / step).round() * step


def _rotate(x, at, s, case):
    """x [n, heads, dim] rotated to the positions `at`, in 64 bits."""
    half = case["rotary"] // 2
    x = x.double()
    c, n = s.cos[at].double()[:, None], s.sin[at].double()[:, None]
    y = x.clone()
    a, b = (slice(0, half), slice(half, 2 * half)) if case["style"] == "neox" else (slice(0, 2 * half, 2),
                                                                                     slice(1, 2 * half, 2))
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., b] * c + x[..., a] * n
    return y


def _plain_append(s):
    case = s.case
    page, dk, dv = case["page"], _padded(case["head_dim"]), _padded(case["v_head_dim"])
    starts, pos = s.starts.long(), s.pos.long()
    counts = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), counts, output_size=s.n_rows)
    at = torch.arange(s.n_rows, device="cuda") - starts[seq] + pos[seq]
    q = _rotate(s.q, at, s, case).to(s.q.dtype)
    new = [torch.nn.functional.pad(_rotate(s.k, at, s, case), (0, dk - case["head_dim"])),
           torch.nn.functional.pad(s.v.double(), (0, dv - case["v_head_dim"]))]
    # the touched pages: `most` slots a sequence, unused ones have no rows
    most = (s.max_rows + page - 2) // page + 1
    slot = seq * most + at // page - pos[seq] // page
    first = (pos // page)[:, None] + torch.arange(most, device="cuda")
    used = (first * page < (pos + counts)[:, None]) & (counts > 0)[:, None]
    ids = s.table.long().gather(1, first.clamp(max=s.cols - 1)).view(-1)[used.view(-1)]
    where = torch.cumsum(used.view(-1), 0) - 1
    slot = where[slot]
    held = (pos[:, None] - first * page).clamp(0, page).view(-1)[used.view(-1)]  # tokens that stay in each page
    keep = torch.arange(page, device="cuda") < held[:, None]
    codes = _unpack(s.codes[0, ids], case)
    scales = s.scales[0, ids]
    packed, sizes = [], []
    for x, old, which in ((new[0], codes[0], 0), (new[1], codes[1], 1)):
        size = x.abs().amax(-1)
        size = torch.zeros(len(ids), case["kv_heads"], dtype=torch.float64,
                           device="cuda").scatter_reduce_(0, slot[:, None].expand_as(size), size, "amax")
        before = torch.where((held > 0)[:, None], scales[..., which], 0)
        after = torch.maximum(before, size.float() / MOST_CODE[case["cache"]])
        inverse = torch.where(after > 0, 1 / after.double(), 0)
        grown = old.double() * (before.double() * inverse)[..., None, None]
        grown = torch.where((after > before)[..., None, None], _round(grown, case["cache"]), old.double())
        grown = torch.where(keep[:, None, :, None], grown, 0)
        grown[slot, :, at % page] = _round(x * inverse[slot][..., None], case["cache"])
        packed.append(grown)
        sizes.append(after)
    s.codes[0, ids] = _pack(packed[0], packed[1], case)
    s.scales[0, ids] = torch.stack(sizes, -1)
    # the touched pages as rows
    k, v = (x.float() * y[..., None, None] for x, y in zip(packed, sizes))
    back = s.back_starts.long()
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), back[1:] - back[:-1], output_size=s.n_back)
    off = torch.arange(s.n_back, device="cuda") - back[seq]
    slot = where[seq * most + off // page]
    return {"q": q, "k": k[slot, :, off % page, :case["head_dim"]], "v": v[slot, :, off % page, :case["v_head_dim"]]}


def _plain_attn(s):
    case = s.case
    kvh, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    ids = s.table.long().clamp(min=0)
    k, v = _unpack(s.codes[0][ids], case)  # [seqs, cols, kvh, page, dim]
    scales = s.scales[0][ids]
    k = (k * scales[..., 0, None, None])[..., :case["head_dim"]].transpose(1, 2).flatten(2, 3)
    v = (v * scales[..., 1, None, None])[..., :case["v_head_dim"]].transpose(1, 2).flatten(2, 3)
    starts, pos = s.starts.long(), s.pos.long()
    counts = starts[1:] - starts[:-1]
    i = torch.arange(s.max_rows, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s.n_rows - 1)
    q = s.q.float()[row].view(case["seqs"], s.max_rows, kvh, group, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)
    w = torch.matmul(q * case["head_dim"] ** -0.5, k.transpose(2, 3))
    at, key = (pos[:, None] + i)[..., None], torch.arange(k.shape[2], device="cuda")
    seen = key <= at
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    w = w.view(case["seqs"], kvh, group, s.max_rows, -1)
    w = w.masked_fill_(~seen[:, None, None], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1)
    o = torch.matmul(w.flatten(2, 3), v).view(case["seqs"], kvh, group, s.max_rows, -1) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    live = i < counts[:, None]
    return o[live].to(s.q.dtype)


def _plain_beam(s):
    case = s.case
    x = s.logits.double()
    x = x - x.amax(-1, keepdim=True)
    x = (x - x.exp().sum(-1, keepdim=True).log()).view(case["prompts"], case["beams"], -1)
    x = (x + s.prev.double()[..., None]).flatten(1)
    # a few more than are wanted, put in order: larger first, then the lower index
    at = x.topk(min(2 * case["k"], x.shape[1]), dim=1).indices.sort(1).values
    best = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, best.indices)[:, :case["k"]]
    return {"scores": best.values[:, :case["k"]].float(), "parents": (at // case["vocab"]).int(),
            "tokens": (at % case["vocab"]).int()}


def _plain_fork(s):
    case = s.case
    g, b, page = case["prompts"], case["beams"], case["page"]
    parents, table = s.parents.long().view(g, b), s.table.view(g, b, s.cols)
    lens = s.lens.long()[:, None, None]
    col = torch.arange(s.cols, device="cuda")
    moved = table.gather(1, parents[..., None].expand(-1, -1, s.cols))
    same = parents[:, :, None] == parents[:, None, :]
    part = (s.lens.long() % page != 0)[:, None]
    copies = torch.tril(same, -1).any(-1) & part  # an earlier child has taken the parent's page over
    childless = ~(parents[:, None, :] == torch.arange(b, device="cuda")[:, None]).any(-1)
    order = childless.int().sort(dim=1, descending=True, stable=True).indices
    last = (s.lens.long() // page).clamp(max=s.cols - 1)
    mine = table.gather(2, last[:, None, None].expand(g, b, 1))[..., 0]
    freed = mine.gather(1, order).gather(1, (copies.cumsum(1) - 1).clamp(min=0))
    spare = s.spare.view(g, b)
    s.table_out.copy_(torch.where((col + 1) * page <= lens, moved,
                                  torch.where(col * page < lens, torch.where(copies[..., None], spare[..., None],
                                                                             moved), table)).view(g * b, -1))
    s.spare_out.copy_(torch.where(copies, freed, spare).view(-1))
    src, dst = moved.gather(2, last[:, None, None].expand(g, b, 1))[..., 0][copies].long(), spare[copies].long()
    s.codes[:, dst] = s.codes[:, src]
    s.scales[:, dst] = s.scales[:, src]
    return _fork_out(s)


def _fork_out(s):
    kind = torch.int8 if s.case["cache"] == "int8" else torch.float8_e4m3fn
    return {"table": s.table_out, "spare": s.spare_out, "codes": s.codes.view(kind), "scales": s.scales}


# ---------------------------------------------------------------------------
# the framework's operators

_dev = None


def _device():
    global _dev
    if _dev is None:
        from ditch_amd.hip import Device
        _dev = Device(0)
    return _dev


def _calls(s):
    """The descriptors that a user's program makes once for its buffers."""
    case, dev = s.case, _device()
    c = _State()
    if case["kind"] == "beam":
        c.bytes = dev.beam_select_workspace(case["prompts"], case["beams"], case["vocab"], case["k"])
        c.ws = torch.empty(c.bytes, dtype=torch.uint8, device="cuda")
        return c
    c.pages = dev.kv_pages(s.codes.data_ptr(), s.codes.numel(), s.scales.data_ptr(), s.scales.numel() * 4,
                           case["cache"], s.codes.shape[0], s.codes.shape[1], case["page"], case["kv_heads"],
                           case["head_dim"], case.get("v_head_dim", case["head_dim"]))
    if case["kind"] == "fork":
        return c

    def batch(starts, pos, n_rows, max_rows):
        return dev.kv_batch(s.table.data_ptr(), s.cols, starts.data_ptr(), pos.data_ptr(), case["seqs"], n_rows,
                            max_rows, s.max_len)

    def rows(x):
        return dev.kv_rows(x.data_ptr(), x.numel() * x.element_size(), x.shape[1] * x.shape[2])

    c.batch = batch(s.starts, s.pos, s.n_rows, s.max_rows)
    c.q = rows(s.q)
    if case["kind"] == "attn":
        c.out = rows(s.out)
        c.bytes = dev.kv_pages_attention_workspace(c.pages, c.batch, case["heads"], case["dtype"], case["window"],
                                                   case["sinks"])
        c.ws = torch.empty(max(c.bytes, 1), dtype=torch.uint8, device="cuda")
    else:
        c.back = batch(s.back_starts, s.back_pos, s.n_back, s.max_back)
        c.k, c.v, c.q_out, c.k_out, c.v_out = (rows(x) for x in (s.k, s.v, s.q_out, s.k_out, s.v_out))
        c.rope = dev.kv_rope(s.cos.data_ptr(), s.sin.data_ptr(), s.max_len, case["rotary"] // 2, case["style"])
    torch.cuda.synchronize()
    return c


def _own(s):
    case, dev = s.case, _device()
    if s.calls is None:
        s.calls = _calls(s)
    c = s.calls
    if case["kind"] == "append":
        dev.kv_pages_append(c.pages, 0, c.batch, case["dtype"], c.k, c.v, rope=c.rope, q=c.q, q_out=c.q_out,
                            heads=case["heads"])
        dev.kv_pages_read(c.pages, 0, c.back, "f32", c.k_out, c.v_out)
        return {"q": s.q_out, "k": s.k_out, "v": s.v_out}
    if case["kind"] == "attn":
        dev.kv_pages_attention(c.pages, 0, c.batch, case["dtype"], c.out, c.q, case["heads"],
                               case["head_dim"] ** -0.5, c.ws.data_ptr(), c.bytes, window=case["window"],
                               sinks=case["sinks"])
        return s.out
    if case["kind"] == "beam":
        dev.beam_select(s.scores.data_ptr(), s.parents.data_ptr(), s.tokens.data_ptr(), s.logits.data_ptr(),
                        s.prev.data_ptr(), case["prompts"], case["beams"], case["vocab"], case["k"],
                        c.ws.data_ptr(), c.bytes)
        return {"scores": s.scores, "parents": s.parents, "tokens": s.tokens}
    dev.kv_pages_fork(c.pages, s.table_out.data_ptr(), s.spare_out.data_ptr(), s.table.data_ptr(), s.cols,
                      s.parents.data_ptr(), s.spare.data_ptr(), s.lens.data_ptr(), case["prompts"], case["beams"])
    return _fork_out(s)


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attn": _plain_attn, "beam": _plain_beam, "fork": _plain_fork}[s.case["kind"]](s)


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _decode_table(cache):
    """The values of the 256 codes."""
    if cache == "int8":
        return torch.tensor([float(c - 256 if c > 127 else c) for c in range(256)], dtype=torch.float64, device="cuda")
    got = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = math.nan if e == 15 and m == 7 else (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        got.append(-x if c & 128 else x)
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def _offsets(case):
    """Where in a head's page the code of (token, dim) lies: of the keys, of the values."""
    dk, dv, page = _padded(case["head_dim"]), _padded(case["v_head_dim"]), case["page"]
    t = torch.arange(page, device="cuda")[:, None]
    d = torch.arange(case["head_dim"], device="cuda")
    k = (t // 16 * (dk // 64) + d // 64) * 1024 + d % 64 // 16 * 256 + t % 16 * 16 + d % 16
    d = torch.arange(case["v_head_dim"], device="cuda")
    u = t % 32
    v = (t // 32 * (dv // 32) + d // 32) * 1024 + u % 16 // 4 * 256 + d % 16 * 16 + d % 32 // 16 * 8 + u // 16 * 4 + u % 4
    return k, page * dk + v


def _nearest(y, values):
    """The entry of `values` (ascending) nearest to each y, ties to the even one (every second, counted from zero)."""
    hi = torch.searchsorted(values, y).clamp(1, len(values) - 1)
    a, b = values[hi - 1], values[hi]
    zero = int((values == 0).nonzero()[0])
    down = (y - a < b - y) | ((y - a == b - y) & ((hi - 1 - zero) % 2 == 0))
    return torch.where(down, a, b)


def _exact_append(case, s):
    rows, pos = _rows_pos(case)
    decode, off = _decode_table(case["cache"]), _offsets(case)
    values = decode[~decode.isnan()].unique()
    if case["cache"] == "int8":
        values = values[values >= -127]
    page, most = case["page"], MOST_CODE[case["cache"]]
    half, hd = case["rotary"] // 2, case["head_dim"]
    pair = torch.arange(half, device="cuda")
    a, b = (pair, pair + half) if case["style"] == "neox" else (2 * pair, 2 * pair + 1)
    table = s.table.tolist()
    qs, ks, vs, at = [], [], [], 0
    for i in range(case["seqs"]):
        if not rows[i]:
            continue
        t = torch.arange(pos[i], pos[i] + rows[i], device="cuda")
        z = torch.complex(s.cos[t].double(), s.sin[t].double())[:, None]
        new = []
        for x in (s.q, s.k):
            x = x[at:at + rows[i]].double()
            w = torch.complex(x[..., a], x[..., b]) * z
            x[..., a], x[..., b] = w.real, w.imag
            new.append(x)
        qs.append(new[0])
        got = [[], []]
        for p in range(pos[i] // page, (pos[i] + rows[i] - 1) // page + 1):
            lo, hi = max(pos[i], p * page), min(pos[i] + rows[i], p * page + page)
            for which, x in enumerate((new[1], s.v[at:at + rows[i]].double())):
                x = x[lo - pos[i]:hi - pos[i]]
                old = decode[s.codes[0, table[i][p]].long()[:, off[which]]][:, :lo - p * page].transpose(0, 1)
                was = s.scales[0, table[i][p], :, which] * (1.0 if lo > p * page else 0.0)
                now = torch.maximum(was, x.abs().amax((0, 2)).float() / most)
                d = now.double()[None, :, None]
                if old.shape[0]:
                    old = torch.where((now > was)[None, :, None], _nearest(old * was.double()[None, :, None] / d,
                                                                           values), old)
                got[which] += [old * d, _nearest(x / d, values) * d]
        ks.append(torch.cat(got[0]))
        vs.append(torch.cat(got[1]))
        at += rows[i]
    return {"q": torch.cat(qs), "k": torch.cat(ks), "v": torch.cat(vs)}


def _exact_attn(case, s):
    rows, pos = _rows_pos(case)
    decode, off = _decode_table(case["cache"]), _offsets(case)
    group, scale = case["heads"] // case["kv_heads"], case["head_dim"] ** -0.5
    out, at = [], 0
    for i in range(case["seqs"]):
        if not rows[i]:
            continue
        n = pos[i] + rows[i]
        ids = s.table[i, :-(-n // case["page"])].long()
        first = max(0, pos[i] - case["window"] + 1) if case["window"] else 0
        o = torch.empty(rows[i], case["heads"], case["v_head_dim"], dtype=torch.float64, device="cuda")
        for h in range(case["kv_heads"]):
            raw = s.codes[0, ids, h].long()
            k = (decode[raw[:, off[0]]] * s.scales[0, ids, h, 0].double()[:, None, None]).flatten(0, 1)[:n]
            v = (decode[raw[:, off[1]]] * s.scales[0, ids, h, 1].double()[:, None, None]).flatten(0, 1)[:n]
            key = torch.arange(n, device="cuda")
            some = (key >= first) | (key < case["sinks"])
            k, v, key = k[some], v[some], key[some]
            for r in range(0, rows[i], 256):
                q = s.q[at + r:min(at + r + 256, at + rows[i]), h * group:(h + 1) * group].double()
                t = torch.arange(pos[i] + r, pos[i] + r + len(q), device="cuda")[:, None]
                w = (q.reshape(-1, q.shape[-1]) @ k.T * scale).view(len(q), group, -1)
                hidden = key > t
                if case["window"]:
                    hidden |= (t - key >= case["window"]) & (key >= case["sinks"])
                w = w.masked_fill(hidden[:, None], -math.inf).softmax(-1)
                o[r:r + len(q), h * group:(h + 1) * group] = (w.flatten(0, 1) @ v).view(len(q), group, -1)
        out.append(o)
        at += rows[i]
    return torch.cat(out)


def _exact_beam(case, s):
    scores, parents, tokens = [], [], []
    for i in range(case["prompts"]):
        x = s.logits[i * case["beams"]:(i + 1) * case["beams"]].double().log_softmax(-1) + s.prev[i].double()[:, None]
        best = x.flatten().sort(descending=True, stable=True)
        scores.append(best.values[:case["k"]])
        parents.append(best.indices[:case["k"]].div(case["vocab"], rounding_mode="floor").int())
        tokens.append(best.indices[:case["k"]].remainder(case["vocab"]).int())
    return {"scores": torch.stack(scores), "parents": torch.stack(parents), "tokens": torch.stack(tokens)}


def _exact_fork(case, s):
    """One prompt after the other, one beam after the other."""
    b, page, length = case["beams"], case["page"], case["length"]
    full, part = length // page, length % page > 0
    parents, table, spare = s.parents.tolist(), s.table.tolist(), s.spare.tolist()
    new_table, new_spare = [list(row) for row in table], list(spare)
    for first in range(0, case["prompts"] * b, b):
        mine = [parents[first + c] for c in range(b)]
        free = [table[first + p][full] for p in range(b) if part and p not in mine]
        for c, p in enumerate(mine):
            new_table[first + c][:full] = table[first + p][:full]
            if not part:
                continue
            new_table[first + c][full] = table[first + p][full]
            if p in mine[:c]:
                new_table[first + c][full] = spare[first + c]
                new_spare[first + c] = free.pop(0)
                s.codes[:, spare[first + c]] = s.codes[:, table[first + p][full]]
                s.scales[:, spare[first + c]] = s.scales[:, table[first + p][full]]
    kind = torch.int8 if case["cache"] == "int8" else torch.float8_e4m3fn
    return {"table": _i32(new_table), "spare": _i32(new_spare), "codes": s.codes.view(kind),
            "scales": s.scales.double()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "beam": _exact_beam, "fork": _exact_fork}[case["kind"]](case,
                                                                                                                s)
