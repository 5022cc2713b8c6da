"""More serving operators around a paged key-value cache: norms of query and key
heads with their rotary positions in one pass (and its gradient), the plan of a
step's pages, rows and slots, attention of prompts and single tokens with a
sliding window and sinks, and attention of a batch that shares a prefix.

Each case is one call of one operator. `run` computes it in plain torch
operations, or with `own` through the session API of fercuda_b200.

A cache holds keys and values in pages [pages, kv_heads, page, head_dim]; slot
s of sequence b is row s % page of page table[b, s // page].
"""
import math
import weakref

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_keep = {}   # the one session a serving process has


# ------------------------------------------------------------------ cases

def _norm(name, rows, q_heads, k_heads, head_dim, dtype, sections, width=0, rotary_dim=0, base=10000.0, interleaved=False,
          axis_freqs=False, far=2048, grad=False):
    c = dict(op="norm", rows=rows, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim, dtype=dtype, axes=len(sections),
             width=width or (q_heads + k_heads) * head_dim, rotary_dim=rotary_dim or head_dim, base=base,
             interleaved=interleaved, axis_freqs=axis_freqs, far=far, grad=grad)
    for i in range(4):
        c["section%d" % i] = sections[i] if i < len(sections) else 0
    return dict(c, name=name) if name else c


def _plan(name, batch, page, slots, tokens, running, ended, tight):
    c = dict(op="plan", batch=batch, page=page, slots=slots, tokens=tokens, running=running, ended=ended, tight=tight)
    return dict(c, name=name) if name else c


def _window(name, batch, tokens, slots, heads, kv_heads, head_dim, page, dtype, window, sinks, ragged):
    c = dict(op="window", batch=batch, tokens=tokens, slots=slots, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             page=page, dtype=dtype, window=window, sinks=sinks, ragged=ragged)
    return dict(c, name=name) if name else c


def _prefix(name, batch, prefix, slots, heads, kv_heads, head_dim, page, dtype, ragged):
    c = dict(op="prefix", batch=batch, prefix=prefix, slots=slots, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             page=page, dtype=dtype, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one conversation: 16 query and 16 key heads of 64 in a fused q|k|v row
        _norm("norm rotary one token", 1, 16, 16, 64, "bf16", [32], width=48 * 64, far=100_000),
        # 64 prompts of 512 tokens, grouped heads of 128: the q and k parts of the fused activation
        _norm("norm rotary prompts", 32768, 32, 8, 128, "bf16", [64], width=48 * 128, base=5e5, far=512),
        # training on video tokens with time, height and width axes, an odd number of them: the gradient
        _norm("norm rotary gradient", 10007, 24, 16, 128, "f16", [16, 24, 24], base=1e6, far=2048, grad=True),
        # a decode step of 64 conversations; one in sixteen begins a page
        _plan("plan step", 64, 16, 2048, 1, 1.0, 0.0, False),
        # requests of very different lengths: prompts enter, conversations go on, some have ended, pages run short
        _plan("plan mixed", 1024, 64, 8192, 512, 0.5, 0.1, True),
        # one short conversation, where only latency counts
        _window("window one short", 1, 1, 101, 16, 16, 64, 16, "bf16", 64, 4, False),
        # a decode step of 64 long conversations behind a window
        _window("window step", 64, 1, 8192, 32, 8, 128, 16, "f16", 2048, 4, True),
        # prompts of 1 to 2048 tokens enter behind a window
        _window("window prompts", 16, 2048, 2125, 32, 8, 128, 64, "bf16", 512, 4, True),
        # a piece of one book-length prompt reads all that came before it
        _window("causal long piece", 1, 4001, 32003, 32, 8, 128, 64, "bf16", 0, 0, False),
        # a few drafts of one short conversation
        _prefix("prefix few short", 4, 128, 37, 16, 16, 64, 16, "bf16", True),
        # a decode step of 64 conversations behind one system text
        _prefix("prefix step", 64, 8192, 1024, 32, 8, 128, 16, "bf16", True),
        # 128 questions about one book
        _prefix("prefix long", 128, 65539, 512, 32, 8, 128, 64, "f16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "plan", "window", "window", "window", "prefix", "prefix"])
    if op == "norm":
        dtype = rng.choice(["bf16", "f16", "f32"])
        head_dim = rng.choice([32, 64, 80, 96, 128, 256])
        kv, group = _log(rng, 1, 16), rng.choice([1, 2, 3, 4, 8])
        heads = kv * (group + 1)
        rows = max(1, min(_log(rng, 1, 32768), (1 << 26) // (heads * head_dim * (2 if dtype == "f32" else 1))))
        rot = head_dim if rng.random() < 0.7 else 2 * rng.randint(4, head_dim // 2)
        cuts = sorted(rng.sample(range(1, rot // 2), rng.randint(1, 4) - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [rot // 2])]
        width = heads * head_dim + rng.choice([0, 0, 1, kv]) * head_dim
        return _norm("", rows, kv * group, kv, head_dim, dtype, sections, width, rot, rng.choice([1e4, 5e5, 1e6]),
                     rng.random() < 0.5, rng.random() < 0.3, _log(rng, 64, 1 << 20), rng.random() < 0.5)
    if op == "plan":
        batch, page = _log(rng, 1, 4096), rng.choice([8, 16, 32, 64, 128])
        slots = _log(rng, 64, 8192)
        tokens = 1 if rng.random() < 0.4 else max(1, min(_log(rng, 2, 4096), slots // 2, (1 << 19) // batch))
        return _plan("", batch, page, slots, tokens, rng.choice([0.0, 0.5, 0.9, 1.0]), rng.choice([0.0, 0.1, 0.3]),
                     rng.random() < 0.4)
    head_dim, page = rng.choice([64, 128, 256]), rng.choice([8, 16, 32, 64, 128])
    kv_heads, dtype = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice(["bf16", "f16"])
    heads, row = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), kv_heads * head_dim
    if op == "window":
        batch = _log(rng, 1, 128)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        tokens = max(1, min(tokens, (1 << 20) // (batch * heads)))
        slots = max(tokens + 1, min(_log(rng, 64, 65536), (1 << 27) // (batch * row), (1 << 31) // (batch * heads * tokens)))
        window = 0 if rng.random() < 0.25 else _log(rng, 16, max(17, slots))
        return _window("", batch, tokens, slots, heads, kv_heads, head_dim, page, dtype, window,
                       rng.choice([0, 1, 4, 16, 130]) if window else 0, rng.random() < 0.7)
    batch = _log(rng, 2, 256)
    prefix = max(16, min(_log(rng, 64, 65536), (1 << 26) // row, (1 << 29) // (batch * heads)))
    slots = max(2, min(_log(rng, 2, 4096), (1 << 26) // (batch * row)))
    return _prefix("", batch, prefix, slots, heads, kv_heads, head_dim, page, dtype, rng.random() < 0.7)


# ------------------------------------------------------------------ inputs

def _sections(c):
    return [c["section%d" % i] for i in range(c["axes"])]


def _prepare_norm(c, s, g):
    dt, width = DTYPES[c["dtype"]], (c["q_heads"] + c["k_heads"]) * c["head_dim"]
    # projections: elements of every size, some channels far larger than the others
    scale = torch.exp(torch.randn(c["width"], generator=g, device="cuda"))
    s["x"] = (torch.randn(c["rows"], c["width"], generator=g, device="cuda") * scale).to(dt)
    s["positions"] = torch.randint(0, c["far"], (c["rows"], c["axes"]), generator=g, device="cuda", dtype=torch.int32)
    s["q_gamma"] = 1 + 0.3 * torch.randn(c["head_dim"], generator=g, device="cuda")
    s["k_gamma"] = 1 + 0.3 * torch.randn(c["head_dim"], generator=g, device="cuda")
    s["out"] = torch.zeros_like(s["x"])
    if c["grad"]:
        s["grad"] = torch.randn(c["rows"], width, generator=g, device="cuda").to(dt)
        s["q_gamma_grad"], s["k_gamma_grad"] = torch.zeros_like(s["q_gamma"]), torch.zeros_like(s["k_gamma"])


def _spread(n, g, low, most):
    """The numbers low .. most spread evenly over n places, in a random order: their sum does not go by the order."""
    even = torch.linspace(low, most, n, device="cuda", dtype=torch.float64) if n > 1 else torch.full((n,), float(most), device="cuda")
    return even.round().to(torch.int32)[torch.randperm(n, generator=g, device="cuda")]


def _prepare_plan(c, s, g):
    B, P = c["batch"], c["page"]
    per = -(-c["slots"] // P)
    ended = int(B * c["ended"])
    going = int((B - ended) * c["running"])
    new = B - ended - going
    # running conversations take one token, new ones a prompt, ended ones none
    slots = _spread(ended + going, g, 1, c["slots"] - c["tokens"])
    place = torch.randperm(B, generator=g, device="cuda")
    z = torch.zeros(max(ended, new), dtype=torch.int32, device="cuda")
    s["held"] = ((torch.cat([slots, z[:new]]) + P - 1) // P).to(torch.int32)[place]
    s["lengths"] = torch.cat([z[:ended], slots[ended:], z[:new]])[place]
    s["counts"] = torch.cat([z[:ended], torch.ones_like(slots[ended:]), _spread(new, g, 1, c["tokens"])])[place]
    s["seen"] = s["lengths"] + torch.randint(0, 9, (B,), generator=g, device="cuda", dtype=torch.int32)
    held = int(s["held"].sum())
    want = int(((s["lengths"] + s["counts"] + P - 1) // P - s["held"]).clamp(min=0).sum())
    free = want * 3 // 4 if c["tight"] else want + 5
    pages = B * per + 8   # some belong to somebody else
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    mine = torch.arange(per, device="cuda") < s["held"][:, None]
    s["table"] = torch.full((B, per), -1, dtype=torch.int32, device="cuda")
    s["table"][mine] = order[:held]
    # a ring of the free pages that begins anywhere
    first = int(torch.randint(0, pages, (1,), generator=g, device="cuda"))
    s["free_pages"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["free_pages"][(first + torch.arange(free, device="cuda")) % pages] = order[held: held + free]
    s["free_state"] = torch.tensor([first, free], dtype=torch.int32, device="cuda")
    s["new_held"], s["new_free_state"] = torch.zeros_like(s["held"]), torch.zeros_like(s["free_state"])
    s["offsets"] = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    rows = int(s["counts"].sum()) + 7   # a padded tail; the sum does not go by the seed
    for n in ("sequences", "positions", "slots"):
        s[n] = torch.zeros(rows, dtype=torch.int32, device="cuda")


def _pages(c, g, batch, slots):
    """Two pools of pages and a table over them in a random order, with a few pages that belong to nobody."""
    per = -(-slots // c["page"])
    pages = batch * per + 3
    shape = (pages, c["kv_heads"], c["page"], c["head_dim"])
    make = lambda: torch.empty(shape, dtype=DTYPES[c["dtype"]], device="cuda").normal_(generator=g)  # noqa: E731
    table = torch.randperm(pages, generator=g, device="cuda")[: batch * per].to(torch.int32)
    return make(), make(), table.view(batch, per)


def _lengths(c, g, low, most):
    """Numbers up to `most` for the batch: all alike, or spread out."""
    return _spread(c["batch"], g, low if c["ragged"] else most, most)


def _prepare_window(c, s, g):
    dt = DTYPES[c["dtype"]]
    s["k"], s["v"], s["table"] = _pages(c, g, c["batch"], c["slots"])
    if c["tokens"] == 1:
        s["lengths"] = _lengths(c, g, 1, c["slots"])
        if c["ragged"] and c["batch"] >= 8:
            s["lengths"][-1] = 0   # an empty place in the batch
        rows = c["batch"]
    else:
        new = _lengths(c, g, 1, c["tokens"])
        s["lengths"] = new + _lengths(c, g, 0, c["slots"] - c["tokens"])
        s["offsets"] = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
        rows = int(new.sum()) + 5   # a padded tail of rows belongs to no sequence
    s["q"] = torch.randn(rows, c["heads"] * c["head_dim"], generator=g, device="cuda").to(dt)
    s["q"] *= 2   # scores spread over several units, as trained heads have them
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(rows, c["heads"], device="cuda")


def _prepare_prefix(c, s, g):
    dt = DTYPES[c["dtype"]]
    per = -(-c["prefix"] // c["page"])
    s["k"], s["v"], table = _pages(c, g, 1, c["batch"] * (-(-c["slots"] // c["page"])) * c["page"] + per * c["page"])
    s["prefix_pages"] = table[0, :per].contiguous()
    s["prefix_length"] = torch.tensor([c["prefix"]], dtype=torch.int32, device="cuda")
    s["table"] = table[0, per:].reshape(c["batch"], -1).contiguous()
    s["lengths"] = _lengths(c, g, 1, c["slots"])
    s["q"] = torch.randn(c["batch"], c["heads"] * c["head_dim"], generator=g, device="cuda").to(dt)
    s["q"] *= 2
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(c["batch"], c["heads"], device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    {"norm": _prepare_norm, "plan": _prepare_plan, "window": _prepare_window, "prefix": _prepare_prefix}[case["op"]](
        case, s, g)
    if own:
        _prepare_own(case, s)
    return s


class _Registered:
    """Buffer ids of tensors that the caller owns; they are freed with the state that holds this."""

    def __init__(self, session, ids):
        weakref.finalize(self, _release, session, ids).atexit = False


def _release(session, ids):
    for i in ids:
        session.free(i)


def _prepare_own(c, s):
    """The session, and the tensors registered with it as buffers for as long as the state lives."""
    from fercuda_b200 import capi
    codes = {torch.float32: capi.FER_DTYPE_F32, torch.float16: capi.FER_DTYPE_F16, torch.bfloat16: capi.FER_DTYPE_BF16,
             torch.int32: capi.FER_DTYPE_I32, torch.uint8: capi.FER_DTYPE_U8}
    if "session" not in _keep:
        _keep["session"] = capi.Session(0, pool_bytes=64 << 20)
    session = s["session"] = _keep["session"]
    session.set_stream(torch.cuda.current_stream().cuda_stream)
    size = 0
    if c["op"] == "norm" and c["grad"]:
        size = capi.norm_rotary_grad_workspace_bytes(c["rows"], c["q_heads"] + c["k_heads"], c["head_dim"])
    elif c["op"] == "window":
        size = capi.paged_window_attention_workspace_bytes(s["q"].shape[0], c["batch"], c["heads"], c["kv_heads"],
                                                           c["head_dim"], s["table"].shape[1] * c["page"], c["window"],
                                                           c["sinks"])
    elif c["op"] == "prefix":
        size = capi.paged_prefix_attention_workspace_bytes(c["batch"], c["heads"], c["kv_heads"], c["head_dim"],
                                                           s["table"].shape[1] * c["page"],
                                                           s["prefix_pages"].shape[0] * c["page"])
    if size:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    s["ids"] = ids = {k: session.import_ptr(codes[t.dtype], list(t.shape), t.data_ptr())
                      for k, t in s.items() if isinstance(t, torch.Tensor)}
    s["registered"] = _Registered(session, list(ids.values()))
    ids.setdefault("workspace", 0)
    if "k" in s:
        s["cache"] = capi.paged_cache(ids["k"], ids["v"], ids["table"], ids["lengths"])


# ------------------------------------------------------------------ one pass

def run(s):
    return {"norm": _run_norm, "plan": _run_plan, "window": _run_window, "prefix": _run_prefix}[s["case"]["op"]](s)


def _angles(c, positions):
    """Cosines and sines [rows, 1, pairs] of a row's pairs: the angles in 64 bits."""
    half = c["rotary_dim"] // 2
    sizes = torch.tensor(_sections(c), device="cuda")
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), sizes, output_size=half)
    pair = torch.arange(half, dtype=torch.float64, device="cuda")
    if c["axis_freqs"]:
        starts = sizes.cumsum(0) - sizes
        expo = (pair - starts[axis]) / sizes[axis]
    else:
        expo = pair / half
    angle = positions.double()[:, axis] * c["base"] ** -expo
    return angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]


def _turn(c, x, cos, sin):
    """The heads [rows, heads, head_dim] turned."""
    half = c["rotary_dim"] // 2
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    if c["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, rest], -1)


EPS = 1e-6


def _run_norm(s):
    c = s["case"]
    heads, D = c["q_heads"] + c["k_heads"], c["head_dim"]
    if own:
        ids = s["ids"]
        how = dict(k_heads=c["k_heads"], q_gamma=ids["q_gamma"], k_gamma=ids["k_gamma"], eps=EPS, sections=_sections(c),
                   rotary_dim=c["rotary_dim"], base=c["base"], interleaved=c["interleaved"], axis_freqs=c["axis_freqs"])
        if c["grad"]:
            s["session"].norm_rotary_grad(ids["x"], ids["grad"], ids["out"], ids["positions"], heads, D,
                                          q_gamma_grad=ids["q_gamma_grad"], k_gamma_grad=ids["k_gamma_grad"],
                                          workspace=ids["workspace"], **how)
        else:
            s["session"].norm_rotary(ids["x"], ids["out"], ids["positions"], heads, D, **how)
    else:
        cos, sin = _angles(c, s["positions"])
        x = s["x"][:, : heads * D].float().view(c["rows"], heads, D)
        key = torch.arange(heads, device="cuda")[:, None] >= c["q_heads"]
        gamma = torch.where(key, s["k_gamma"], s["q_gamma"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        if c["grad"]:
            g = _turn(c, s["grad"].float().view(c["rows"], heads, D), cos, -sin)
            unit = x * r
            s["q_gamma_grad"].copy_((g * unit)[:, : c["q_heads"]].sum((0, 1)))
            s["k_gamma_grad"].copy_((g * unit)[:, c["q_heads"]:].sum((0, 1)))
            g = g * gamma
            y = r * (g - unit * (g * unit).mean(-1, keepdim=True))
        else:
            y = _turn(c, x * r * gamma, cos, sin)
        s["out"][:, : heads * D] = y.reshape(c["rows"], -1).to(s["out"].dtype)
    return {n: s[n] for n in (("out", "q_gamma_grad", "k_gamma_grad") if c["grad"] else ("out",))}


def _run_plan(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].paged_plan(ids["table"], ids["lengths"], ids["counts"], ids["held"], ids["free_pages"],
                                ids["free_state"], ids["offsets"], page_size=c["page"], new_held=ids["new_held"],
                                new_free_state=ids["new_free_state"], sequences=ids["sequences"],
                                positions=ids["positions"], seen=ids["seen"], slots=ids["slots"])
    else:
        P, ring = c["page"], s["free_pages"].shape[0]
        n, held = s["lengths"].long(), s["held"].long()
        first, free = s["free_state"].long().unbind()
        keep, need = (n + P - 1) // P, (n + s["counts"] + P - 1) // P
        ask = (need - held).clamp(min=0)
        granted = (ask == 0) | (ask.cumsum(0) <= free)
        count = torch.where(granted, s["counts"].long(), 0)
        new = torch.where(granted, need, torch.minimum(held, keep))
        take, give = (new - held).clamp(min=0), (held - new).clamp(min=0)
        at = torch.arange(s["table"].shape[1], device="cuda")
        # pages leave the ring at its beginning and come back behind its end
        back = (at >= new[:, None]) & (at < held[:, None])
        rank = (give.cumsum(0) - give - new)[:, None] + at
        s["free_pages"][((first + free + rank) % ring)[back]] = s["table"][back]
        gets = (at >= held[:, None]) & (at < new[:, None])
        rank = (take.cumsum(0) - take - held)[:, None] + at
        s["table"][gets] = s["free_pages"][((first + rank) % ring)[gets]]
        s["new_held"].copy_(new)
        s["new_free_state"].copy_(torch.stack([(first + take.sum()) % ring, free - take.sum() + give.sum()]))
        s["offsets"][1:] = count.cumsum(0).to(torch.int32)
        ends = s["offsets"].long()[1:]
        row = torch.arange(s["slots"].shape[0], device="cuda")
        seq = torch.searchsorted(ends, row, right=True)   # behind the last sequence: batch
        on, seq = seq < c["batch"], seq.clamp(max=c["batch"] - 1)
        i = row - ends[seq] + count[seq]
        slot = n[seq] + torch.where(on, i, 0)
        page = s["table"].long()[seq, (slot // P).clamp(max=s["table"].shape[1] - 1)]
        s["sequences"].copy_(torch.where(on, seq, -1))
        s["positions"].copy_(torch.where(on, s["seen"].long()[seq] + i, 0))
        s["slots"].copy_(torch.where(on, page * P + slot % P, -1))
    return {n: s[n] for n in ("table", "free_pages", "new_held", "new_free_state", "offsets", "sequences", "positions",
                              "slots")}


def _gather(pages, table):
    """The rows of each sequence in slot order, in 32 bits: [batch, kv_heads, slots, head_dim]."""
    return pages[table.long()].transpose(1, 2).flatten(2, 3).float()


def _softmax(score, seen):
    """Probabilities and log of the sum of exp over the visible slots; rows that see nothing give 0 and -inf."""
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    return e.div_(torch.where(total == 0, 1.0, total)), (top + total.log())[..., 0]


def _run_window(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].paged_window_attention(s["cache"], ids["q"], ids["out"], c["heads"], c["window"], c["sinks"],
                                            offsets=0 if c["tokens"] == 1 else ids["offsets"], lse=ids["lse"],
                                            workspace=ids["workspace"])
    else:
        B, H, D, group, T = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], c["tokens"]
        k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
        n = s["lengths"].long()
        if T == 1:
            seq, at, new = torch.arange(B, device="cuda"), torch.zeros(B, dtype=torch.int64, device="cuda"), n.new_ones(B)
        else:
            new = (s["offsets"][1:] - s["offsets"][:-1]).long()
            row = torch.arange(s["q"].shape[0], device="cuda")
            seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)   # behind the last sequence: batch
            seq = seq[seq < B]
            at = row[: seq.shape[0]] - s["offsets"].long()[seq]
        # the rows side by side, one sequence each: [batch, tokens, heads, head_dim]
        q = torch.zeros(B, T, c["heads"], D, device="cuda")
        q[seq, at] = s["q"][: seq.shape[0]].float().view(-1, c["heads"], D)
        q = q.view(B, T, H, group, D).permute(0, 2, 3, 1, 4).reshape(B, H, group * T, D)
        slot = torch.arange(k.shape[2], device="cuda")
        place = (n - new)[:, None] + torch.arange(T, device="cuda")   # the slot of each row
        seen = slot <= place[:, :, None]
        if c["window"]:
            seen &= (slot > place[:, :, None] - c["window"]) | (slot < c["sinks"])
        score = (q @ k.transpose(2, 3)).div_(math.sqrt(D)).view(B, H, group, T, -1)
        p, lse = _softmax(score, seen[:, None, None])
        held = (slot < n[:, None])[:, None, :, None]
        out = p.view(B, H, group * T, -1) @ v.masked_fill(~held, 0.0)
        out = out.view(B, H, group, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, -1)
        s["out"][: seq.shape[0]] = out[seq, at].to(s["out"].dtype)
        s["lse"][: seq.shape[0]] = lse.permute(0, 3, 1, 2).reshape(B, T, -1)[seq, at]
    return {"out": s["out"], "lse": s["lse"]}


def _run_prefix(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].paged_prefix_attention(s["cache"], ids["prefix_pages"], ids["prefix_length"], ids["q"], ids["out"],
                                            c["heads"], lse=ids["lse"], workspace=ids["workspace"])
    else:
        B, H, D, group = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
        pk, pv = _gather(s["k"], s["prefix_pages"][None])[0], _gather(s["v"], s["prefix_pages"][None])[0]
        k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
        shared = torch.arange(pk.shape[1], device="cuda") < s["prefix_length"]
        held = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]
        q = s["q"].float().view(B, H, group, D)
        side = q.transpose(0, 1).reshape(H, B * group, D)   # all of a key head's queries
        first = (side @ pk.transpose(1, 2)).view(H, B, group, -1).transpose(0, 1)
        score = torch.cat([first, q @ k.transpose(2, 3)], -1).div_(math.sqrt(D))
        seen = torch.cat([shared[None].expand(B, -1), held], -1)
        p, lse = _softmax(score, seen[:, None, None])
        first = p[..., : pk.shape[1]].transpose(0, 1).reshape(H, B * group, -1) @ pv.masked_fill(~shared[:, None], 0.0)
        out = first.view(H, B, group, D).transpose(0, 1) + \
            p[..., pk.shape[1]:] @ v.masked_fill(~held[:, None, :, None], 0.0)
        s["out"].copy_(out.reshape(B, -1))
        s["lse"].copy_(lse.reshape(B, -1))
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------ what a pass cannot do without

def _visible(c, place):
    """Slots that a row in slot `place` sees."""
    if not c["window"]:
        return place + 1
    near = min(place + 1, c["window"])
    return near + min(c["sinks"], place + 1 - near)


def work(c):
    size = 4 if c.get("dtype") == "f32" else 2
    if c["op"] == "norm":
        n = c["rows"] * (c["q_heads"] + c["k_heads"]) * c["head_dim"]
        moved = (3 if c["grad"] else 2) * n * size + 4 * c["rows"] * c["axes"] + 8 * c["head_dim"]
        return {"bytes": moved + (8 * c["head_dim"] if c["grad"] else 0), "flops": (14 if c["grad"] else 7) * n}
    if c["op"] == "plan":
        per = c["running"] + (1 - c["running"]) * (c["tokens"] + 1) / 2
        rows = c["batch"] * (1 - c["ended"]) * per * (0.75 if c["tight"] else 1)
        pages = c["batch"] * ((1 - c["ended"]) * (1 - c["running"]) * max(1, c["tokens"] / 2 / c["page"]) +
                              c["ended"] * c["slots"] / 2 / c["page"])
        return {"bytes": 24 * c["batch"] + 12 * rows + 8 * pages, "flops": 0}
    row = c["kv_heads"] * c["head_dim"] * 2 * size     # one slot's key and value over all heads
    spread = c["ragged"] and c["batch"] > 1
    heads, D, B = c["heads"], c["head_dim"], c["batch"]
    if c["op"] == "window":
        new = (c["tokens"] + 1) / 2 if spread and c["tokens"] > 1 else c["tokens"]
        before = (c["slots"] - c["tokens"]) / (2 if spread else 1)
        if c["tokens"] == 1:   # the mean over even lengths
            steps = [(i + 0.5) / 64 * c["slots"] - 1 for i in range(64)] if spread else [c["slots"] - 1]
        else:
            steps = [before + (i + 0.5) / 64 * new for i in range(64)]
        seen = sum(_visible(c, p) for p in steps) / len(steps)
        slots = seen if c["tokens"] == 1 else min(before + new, seen + new)
        return {"bytes": B * (slots * row + new * heads * (2 * D * size + 4)), "flops": 4 * B * new * seen * heads * D}
    slots = B * ((c["slots"] + 1) / 2 if spread else c["slots"])
    return {"bytes": (c["prefix"] + slots) * row + B * heads * (2 * D * size + 4),
            "flops": 4 * heads * D * (B * c["prefix"] + slots)}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "plan": _exact_plan, "window": _exact_window, "prefix": _exact_prefix}[case["op"]](case, s)


def _exact_norm(c, s):
    heads, D, half = c["q_heads"] + c["k_heads"], c["head_dim"], c["rotary_dim"] // 2
    out = s["out"].double()
    sums = {"q_gamma_grad": torch.zeros(D, dtype=torch.float64, device="cuda"),
            "k_gamma_grad": torch.zeros(D, dtype=torch.float64, device="cuda")}
    freq, axis, i = [], [], 0
    for a in range(c["axes"]):
        for j in range(c["section%d" % a]):
            freq.append(math.exp(-math.log(c["base"]) * (j / c["section%d" % a] if c["axis_freqs"] else i / half)))
            axis.append(a)
            i += 1
    theta = s["positions"].double()[:, axis] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones_like(theta), -theta if c["grad"] else theta)
    pairs = torch.arange(half, device="cuda")
    u, w = (2 * pairs, 2 * pairs + 1) if c["interleaved"] else (pairs, pairs + half)

    def rotated(z):
        z = z.clone()
        t = torch.complex(z[:, u], z[:, w]) * turn
        z[:, u], z[:, w] = t.real, t.imag
        return z

    for h in range(heads):   # head by head
        x = s["x"][:, h * D: (h + 1) * D].double()
        name = "k" if h >= c["q_heads"] else "q"
        gamma = s[name + "_gamma"].double()
        size = ((x ** 2).sum(1, keepdim=True) / D + EPS) ** 0.5
        if c["grad"]:
            g = rotated(s["grad"][:, h * D: (h + 1) * D].double())
            sums[name + "_gamma_grad"] += (g * x / size).sum(0)
            g = g * gamma
            out[:, h * D: (h + 1) * D] = g / size - x * (g * x).sum(1, keepdim=True) / (D * size ** 3)
        else:
            out[:, h * D: (h + 1) * D] = rotated(x / size * gamma)
    return dict(out=out, **sums) if c["grad"] else dict(out=out)


def _exact_plan(c, s):
    return None   # whole numbers


def _exact_window(c, s):
    B, H, D, group = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    if work(c)["flops"] > 3e11:   # half a minute and more in 64 bits
        return None
    out, lse = s["out"].double(), s["lse"].double()
    off = s["offsets"].tolist() if c["tokens"] > 1 else list(range(B + 1))
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, : -(-n // c["page"])].long()
        for h in range(H):
            k = s["k"][pages, h].reshape(-1, D)[:n].double()
            v = s["v"][pages, h].reshape(-1, D)[:n].double()
            for lo in range(off[b], off[b + 1], 512):   # rows lo .. hi in slots first ..
                hi = min(off[b + 1], lo + 512)
                cols = slice(h * group, (h + 1) * group)
                if n == 0:
                    out.view(-1, c["heads"], D)[lo: hi, cols] = 0.0
                    lse[lo: hi, cols] = -math.inf
                    continue
                first = n - off[b + 1] + lo
                q = s["q"].view(-1, c["heads"], D)[lo: hi, cols].double()
                z = torch.einsum("tgd,sd->tgs", q, k) * D ** -0.5
                back = torch.arange(first, first + hi - lo, device="cuda")[:, None] - torch.arange(n, device="cuda")
                hidden = back < 0
                if c["window"]:
                    hidden |= (back >= c["window"]) & (torch.arange(n, device="cuda") >= c["sinks"])
                z[hidden[:, None].expand_as(z)] = -math.inf
                lse[lo: hi, cols] = torch.logsumexp(z, 2)
                out.view(-1, c["heads"], D)[lo: hi, cols] = torch.einsum("tgs,sd->tgd", torch.softmax(z, 2), v)
    return {"out": out, "lse": lse}


def _exact_prefix(c, s):
    B, H, D, group = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    if work(c)["flops"] > 3e11:
        return None
    out = torch.zeros(B, c["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, c["heads"], dtype=torch.float64, device="cuda")
    shared = s["prefix_pages"].long()
    for h in range(H):
        pk = s["k"][shared, h].reshape(-1, D)[: c["prefix"]].double()
        pv = s["v"][shared, h].reshape(-1, D)[: c["prefix"]].double()
        for b, n in enumerate(s["lengths"].tolist()):
            pages = s["table"][b, : -(-n // c["page"])].long()
            k = torch.cat([pk, s["k"][pages, h].reshape(-1, D)[:n].double()])
            v = torch.cat([pv, s["v"][pages, h].reshape(-1, D)[:n].double()])
            cols = slice(h * group, (h + 1) * group)
            z = torch.mm(s["q"].view(B, c["heads"], D)[b, cols].double(), k.t()) * D ** -0.5
            lse[b, cols] = torch.logsumexp(z, 1)
            out[b, cols] = torch.mm(torch.softmax(z, 1), v)
    return {"out": out.view(B, -1), "lse": lse}
