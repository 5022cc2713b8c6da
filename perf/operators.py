"""The serving operators around a paged key-value cache: rotary positions with
several axes, the store of new keys and values into pages, attention of one
new token over the pages, and eviction by accumulated attention weight.

Each case is one call of one operator. `run` computes it in plain torch
operations, or with `own` through the session API of fercuda_b200.

A cache holds keys and values in pages [pages, kv_heads, page, head_dim]; slot
s of sequence b is row s % page of page table[b, s // page]. For every slot it
may keep the attention weight summed so far and the position of its token,
both [batch, kv_heads, slots].
"""
import math
import weakref

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_keep = {}   # the one session a serving process has


# ------------------------------------------------------------------ cases

def _rotary(name, rows, heads, head_dim, dtype, sections, width=0, rotary_dim=0, base=10000.0, interleaved=False,
            axis_freqs=False, inverse=False, far=0):
    c = dict(op="rotary", rows=rows, heads=heads, head_dim=head_dim, dtype=dtype, axes=len(sections),
             width=width or heads * head_dim, rotary_dim=rotary_dim or head_dim, base=base, interleaved=interleaved,
             axis_freqs=axis_freqs, inverse=inverse, far=far)
    for i in range(4):
        c["section%d" % i] = sections[i] if i < len(sections) else 0
    return dict(c, name=name) if name else c


def _store(name, batch, tokens, kv_heads, head_dim, page, dtype, ragged, held):
    c = dict(op="store", batch=batch, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
             ragged=ragged, held=held)
    return dict(c, name=name) if name else c


def _attention(name, batch, slots, heads, kv_heads, head_dim, page, dtype, ragged, weights):
    c = dict(op="attention", batch=batch, slots=slots, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
             dtype=dtype, ragged=ragged, weights=weights)
    return dict(c, name=name) if name else c


def _evict(name, batch, slots, kv_heads, head_dim, page, dtype, budget, recent, ragged, shuffled):
    c = dict(op="evict", batch=batch, slots=slots, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
             budget=budget, recent=recent, ragged=ragged, shuffled=shuffled)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one conversation: 16 query and 16 key heads of 64 in a fused q|k|v row
        _rotary("rotary one token", 1, 32, 64, "bf16", [32], width=48 * 64, far=100_000),
        # 64 prompts of 512 tokens, the q and k thirds of the fused activation
        _rotary("rotary prompts", 32768, 32, 64, "bf16", [32], width=48 * 64, far=512),
        # the gradient of video tokens with time, height and width axes, an odd number of them
        _rotary("rotary video gradient", 10007, 40, 128, "f16", [16, 24, 24], base=1e6, inverse=True, far=2048),
        # a decode step of 64 conversations writes one key and value row each
        _store("store step", 64, 1, 16, 64, 16, "bf16", False, 700),
        # 37 prompts of 1 to 2048 tokens enter the pages behind a shared system text
        _store("store prompts", 37, 2048, 8, 128, 64, "f16", True, 77),
        # one short conversation, where only latency counts
        _attention("attention one short", 1, 101, 16, 16, 64, 16, "bf16", False, False),
        # a decode step of 64 conversations of about a thousand tokens, every head its own keys
        _attention("attention step", 64, 1024, 16, 16, 64, 16, "bf16", True, False),
        # grouped heads, very different lengths and an empty place in the batch, weights summed for eviction
        _attention("attention grouped weights", 33, 8192, 32, 8, 128, 16, "f16", True, True),
        # one very long context
        _attention("attention long", 1, 131071, 64, 8, 128, 64, "bf16", False, False),
        # weights over one book-length context
        _attention("attention long weights", 2, 40003, 16, 4, 128, 32, "bf16", False, True),
        # each step a full cache gives up one slot per head
        _evict("evict step", 64, 513, 16, 64, 16, "bf16", 512, 64, False, True),
        # long prompts are cut down to 4096 slots before decoding starts
        _evict("evict prompts", 4, 32768, 8, 128, 64, "bf16", 4096, 256, True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "store", "attention", "attention", "evict"])
    if op == "rotary":
        dtype = rng.choice(["bf16", "f16", "f32"])
        head_dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = _log(rng, 1, 64)
        rows = min(_log(rng, 1, 32768), (1 << 26) // (heads * head_dim * (2 if dtype == "f32" else 1)))
        rot = head_dim if rng.random() < 0.7 else 2 * rng.randint(4, head_dim // 2)
        cuts = sorted(rng.sample(range(1, rot // 2), rng.randint(1, 4) - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [rot // 2])]
        width = heads * head_dim + (rng.choice([0, 0, 1, 3]) * head_dim)
        return _rotary("", rows, heads, head_dim, dtype, sections, width, rot, rng.choice([1e4, 5e5, 1e6]),
                       rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.3, _log(rng, 64, 1 << 20))
    head_dim, page = rng.choice([64, 128, 256]), rng.choice([8, 16, 32, 64, 128])
    kv_heads, dtype = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice(["bf16", "f16"])
    ragged, row = rng.random() < 0.7, kv_heads * head_dim
    if op == "store":
        batch = _log(rng, 1, 128)
        tokens = min(_log(rng, 1, 4096), max(1, (1 << 25) // (batch * row)))
        held = min(_log(rng, 1, 2000), max(1, (1 << 26) // (batch * row)))
        return _store("", batch, tokens, kv_heads, head_dim, page, dtype, ragged, held)
    batch = _log(rng, 1, 256)
    slots = max(2, min(_log(rng, 2, 131072), (1 << 27) // (batch * row)))
    if op == "attention":
        slots = max(2, min(slots, (1 << 27) // (batch * kv_heads * 16)))
        return _attention("", batch, slots, kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), kv_heads, head_dim,
                          page, dtype, ragged, rng.random() < 0.5)
    slots = min(slots, 32768)
    budget = slots - 1 if rng.random() < 0.3 else max(1, int(slots * rng.uniform(0.1, 0.9)))
    return _evict("", batch, slots, kv_heads, head_dim, page, dtype, budget, rng.randint(0, budget), ragged,
                  rng.random() < 0.5)


# ------------------------------------------------------------------ inputs

def _lengths(case, g, most):
    """Lengths up to `most`: all alike, or spread out with the longest and (in batches of 8 and more) an empty one among them."""
    n = torch.full((case["batch"],), most, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        n = torch.randint(1, most + 1, (case["batch"],), generator=g, device="cuda", dtype=torch.int32)
        n[0] = most
        if case["batch"] >= 8 and case["op"] != "store":
            n[-1] = 0
    return n


def _pages(case, g, slots):
    """Two pools of pages and a table over them in a random order, with a few pages that belong to nobody."""
    per = -(-slots // case["page"])
    pages = case["batch"] * per + 3
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    make = lambda: torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=g)  # noqa: E731
    table = torch.randperm(pages, generator=g, device="cuda")[: case["batch"] * per].to(torch.int32)
    return make(), make(), table.view(case["batch"], per)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "rotary":
        dt = DTYPES[case["dtype"]]
        s["x"] = torch.randn(case["rows"], case["width"], generator=g, device="cuda").to(dt)
        s["out"] = torch.zeros_like(s["x"])
        s["positions"] = torch.randint(0, case["far"], (case["rows"], case["axes"]), generator=g, device="cuda",
                                       dtype=torch.int32)
    else:
        _prepare_cache(case, s, g)
    if own:
        _prepare_own(case, s)
    return s


def _prepare_cache(case, s, g):
    dt, B, H = DTYPES[case["dtype"]], case["batch"], case["kv_heads"]
    slots = case["held"] + case["tokens"] if case["op"] == "store" else case["slots"]
    s["k"], s["v"], s["table"] = _pages(case, g, slots)
    slots = s["table"].shape[1] * case["page"]
    s["weights"] = torch.zeros(B, H, slots, device="cuda")
    s["positions"] = torch.zeros(B, H, slots, dtype=torch.int32, device="cuda")
    if case["op"] == "store":
        s["lengths"] = torch.full((B,), case["held"], dtype=torch.int32, device="cuda")
        s["seen"] = s["lengths"] + torch.randint(0, 9, (B,), generator=g, device="cuda", dtype=torch.int32)
        new = _lengths(case, g, case["tokens"])
        s["offsets"] = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
        # one fused k|v activation; a padded tail of rows belongs to no sequence
        rows = B if case["tokens"] == 1 else int(new.sum()) + 5
        s["rows"] = torch.randn(rows, 2 * H * case["head_dim"], generator=g, device="cuda").to(dt)
        s["new_lengths"], s["new_seen"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["lengths"])
        s["weights"].uniform_(generator=g)
        return
    s["lengths"] = _lengths(case, g, case["slots"])
    if case["op"] == "attention":
        s["q"] = torch.randn(B, case["heads"] * case["head_dim"], generator=g, device="cuda").to(dt)
        s["q"] *= 2   # scores spread over several units, as trained heads have them
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(B, case["heads"], device="cuda")
        return
    # sums of attention weights have a long tail, and many that underflowed to the same zero
    s["weights"].log_normal_(0.0, 2.0, generator=g)
    s["weights"][torch.rand(s["weights"].shape, generator=g, device="cuda") < 0.1] = 0.0
    if case["shuffled"]:   # earlier evictions have mixed the order of positions
        noise = torch.rand(s["weights"].shape, generator=g, device="cuda")
        noise.masked_fill_(torch.arange(slots, device="cuda") >= s["lengths"][:, None, None], 2.0)
        s["positions"] += noise.argsort(-1).to(torch.int32)
    else:
        s["positions"] += torch.arange(slots, dtype=torch.int32, device="cuda")
    s["seen"] = s["lengths"].clone()
    s["new_lengths"], s["new_weights"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["weights"])
    s["new_positions"] = torch.zeros_like(s["positions"])


class _Registered:
    """Buffer ids of tensors that the caller owns; they are freed with the state that holds this."""

    def __init__(self, session, ids):
        weakref.finalize(self, _release, session, ids).atexit = False


def _release(session, ids):
    for i in ids:
        session.free(i)


def _prepare_own(case, s):
    """The session, and the tensors registered with it as buffers for as long as the state lives."""
    from fercuda_b200 import capi
    codes = {torch.float32: capi.FER_DTYPE_F32, torch.float16: capi.FER_DTYPE_F16, torch.bfloat16: capi.FER_DTYPE_BF16,
             torch.int32: capi.FER_DTYPE_I32, torch.uint8: capi.FER_DTYPE_U8}
    if "session" not in _keep:
        _keep["session"] = capi.Session(0, pool_bytes=64 << 20)
    session = s["session"] = _keep["session"]
    session.set_stream(torch.cuda.current_stream().cuda_stream)
    size = 0
    if case["op"] == "attention":
        size = capi.paged_attention_workspace_bytes(case["batch"], case["heads"], case["kv_heads"], case["head_dim"],
                                                    s["table"].shape[1] * case["page"], case["weights"])
    elif case["op"] == "evict":
        size = capi.paged_evict_workspace_bytes(case["batch"], case["kv_heads"], s["table"].shape[1] * case["page"],
                                                case["budget"])
    if size:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    s["ids"] = ids = {k: session.import_ptr(codes[t.dtype], list(t.shape), t.data_ptr())
                      for k, t in s.items() if isinstance(t, torch.Tensor)}
    s["registered"] = _Registered(session, list(ids.values()))
    ids.setdefault("workspace", 0)
    if case["op"] != "rotary":
        s["cache"] = capi.paged_cache(ids["k"], ids["v"], ids["table"], ids["lengths"])


# ------------------------------------------------------------------ one pass

def run(s):
    return {"rotary": _run_rotary, "store": _run_store, "attention": _run_attention,
            "evict": _run_evict}[s["case"]["op"]](s)


def _sections(c):
    return [c["section%d" % i] for i in range(c["axes"])]


def _run_rotary(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].rotary(ids["x"], ids["out"], ids["positions"], c["heads"], c["head_dim"], sections=_sections(c),
                            rotary_dim=c["rotary_dim"], base=c["base"], interleaved=c["interleaved"],
                            axis_freqs=c["axis_freqs"], inverse=c["inverse"])
        return s["out"]
    half = c["rotary_dim"] // 2
    # the axis of each pair, the pair's exponent, and its angle in 64 bits
    sizes = torch.tensor(_sections(c), device="cuda")
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), sizes, output_size=half)
    pair = torch.arange(half, dtype=torch.float64, device="cuda")
    if c["axis_freqs"]:
        starts = sizes.cumsum(0) - sizes
        expo = (pair - starts[axis]) / sizes[axis]
    else:
        expo = pair / half
    angle = s["positions"].double()[:, axis] * c["base"] ** -expo
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    if c["inverse"]:
        sin = -sin
    x = s["x"][:, : c["heads"] * c["head_dim"]].float().view(c["rows"], c["heads"], c["head_dim"])
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    if c["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    y = torch.cat([y, rest], -1).view(c["rows"], -1)
    s["out"][:, : y.shape[1]] = y.to(s["out"].dtype)
    return s["out"]


def _run_store(s):
    c = s["case"]
    H, D = c["kv_heads"], c["head_dim"]
    if own:
        ids = s["ids"]
        s["session"].paged_store(s["cache"], ids["rows"], ids["rows"], k_col=0, v_col=H * D,
                                 offsets=0 if c["tokens"] == 1 else ids["offsets"], new_lengths=ids["new_lengths"],
                                 weights=ids["weights"], positions=ids["positions"], seen=ids["seen"],
                                 new_seen=ids["new_seen"])
    else:
        row = torch.arange(s["rows"].shape[0], device="cuda")
        seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)   # behind the last sequence: batch
        row, seq = row[seq < c["batch"]], seq[seq < c["batch"]]
        at = row - s["offsets"].long()[seq]
        slot = s["lengths"].long()[seq] + at
        page = s["table"].long()[seq, slot // c["page"]]
        kv = s["rows"].view(-1, 2, H, D)
        s["k"][page, :, slot % c["page"]] = kv[row, 0]
        s["v"][page, :, slot % c["page"]] = kv[row, 1]
        s["weights"][seq, :, slot] = 0.0
        s["positions"][seq, :, slot] = (s["seen"].long()[seq] + at).to(torch.int32)[:, None]
        new = s["offsets"][1:] - s["offsets"][:-1]
        s["new_lengths"].copy_(s["lengths"] + new)
        s["new_seen"].copy_(s["seen"] + new)
    return {n: s[n] for n in ("k", "v", "weights", "positions", "new_lengths", "new_seen")}


def _gather(pages, table):
    """The rows of each sequence in slot order, in 32 bits: [batch, kv_heads, slots, head_dim]."""
    return pages[table.long()].transpose(1, 2).flatten(2, 3).float()


def _run_attention(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].paged_attention(s["cache"], ids["q"], ids["out"], c["heads"], lse=ids["lse"],
                                     weights=ids["weights"] if c["weights"] else 0, workspace=ids["workspace"])
    else:
        B, H, D, group = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
        k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
        held = (torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None])[:, None, None, :]
        q = s["q"].float().view(B, H, group, D)
        score = (q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill(~held, -math.inf)
        some = (s["lengths"] > 0)[:, None, None, None]
        top = torch.where(some, score.amax(-1, keepdim=True), 0.0)
        e = torch.exp(score - top)
        total = e.sum(-1, keepdim=True)
        p = torch.where(some, e / total, 0.0)
        s["out"].copy_((p @ v.masked_fill(~held.transpose(2, 3), 0.0)).view(B, -1))
        s["lse"].copy_((top + total.log()).view(B, -1))
        if c["weights"]:
            s["weights"] += p.sum(2)
    return {n: s[n] for n in (("out", "lse", "weights") if c["weights"] else ("out", "lse"))}


def _run_evict(s):
    c = s["case"]
    if own:
        ids = s["ids"]
        s["session"].paged_evict(s["cache"], c["budget"], c["recent"], ids["weights"], ids["positions"], ids["seen"],
                                 new_lengths=ids["new_lengths"], new_weights=ids["new_weights"],
                                 new_positions=ids["new_positions"], workspace=ids["workspace"])
    else:
        slot = torch.arange(s["weights"].shape[2], device="cuda")
        n = s["lengths"][:, None, None]
        valid = slot < n
        late = s["positions"] >= s["seen"][:, None, None] - c["recent"]
        value = torch.where(valid, torch.where(late, math.inf, s["weights"]), -math.inf)
        order = value.sort(dim=-1, descending=True, stable=True).indices
        rank = torch.empty_like(order).scatter_(2, order, slot.expand_as(order).contiguous())
        kept = valid & (rank < c["budget"])
        stay = kept & (slot < c["budget"])
        s["new_weights"].copy_(torch.where(stay, s["weights"], s["new_weights"]))
        s["new_positions"].copy_(torch.where(stay, s["positions"], s["new_positions"]))
        # the i-th kept slot behind the budget moves to the i-th free slot before it
        b, h, to = (valid & ~kept & (slot < c["budget"])).nonzero(as_tuple=True)
        _, _, at = (kept & (slot >= c["budget"])).nonzero(as_tuple=True)
        s["new_weights"][b, h, to] = s["weights"][b, h, at]
        s["new_positions"][b, h, to] = s["positions"][b, h, at]
        table, page = s["table"].long(), c["page"]
        at_page, to_page = table[b, at // page], table[b, to // page]
        s["k"][to_page, h, to % page] = s["k"][at_page, h, at % page]
        s["v"][to_page, h, to % page] = s["v"][at_page, h, at % page]
        s["new_lengths"].copy_(s["lengths"].clamp(max=c["budget"]))
    return {n: s[n] for n in ("k", "v", "new_weights", "new_positions", "new_lengths")}


# ------------------------------------------------------------------ what a pass cannot do without

def _mean_length(c, most):
    return (most + 1) / 2 if c["ragged"] and c["batch"] > 1 else most


def work(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rotary":
        n = c["rows"] * c["heads"] * c["head_dim"]
        return {"bytes": 2 * n * size + 4 * c["rows"] * c["axes"], "flops": 3 * n}
    row = c["kv_heads"] * c["head_dim"] * 2 * size     # one slot's key and value over all heads
    if c["op"] == "store":
        tokens = c["batch"] * _mean_length(c, c["tokens"])
        return {"bytes": tokens * (2 * row + 8 * c["kv_heads"]) + 20 * c["batch"], "flops": 0}
    slots = c["batch"] * _mean_length(c, c["slots"])
    if c["op"] == "attention":
        bytes_ = slots * (row + 4 / c["page"]) + c["batch"] * c["heads"] * (2 * c["head_dim"] * size + 4)
        if c["weights"]:
            bytes_ += slots * c["kv_heads"] * 8
        return {"bytes": bytes_, "flops": 4 * slots * c["heads"] * c["head_dim"]}
    n, kept = _mean_length(c, c["slots"]), min(c["budget"], _mean_length(c, c["slots"]))
    behind = max(0.0, n - kept)
    recent = min(c["recent"], behind if not c["shuffled"] else 0)
    share = behind * kept / n if c["shuffled"] else recent + (kept - recent) * (behind - recent) / max(1, n - recent)
    return {"bytes": c["batch"] * (c["kv_heads"] * 8 * (n + kept) + share * 2 * row) + 12 * c["batch"], "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "store": _exact_store, "attention": _exact_attention,
            "evict": _exact_evict}[case["op"]](case, s)


def _exact_rotary(c, s):
    y = s["out"].double()
    half, inner = c["rotary_dim"] // 2, 0
    x = s["x"].double()
    for a in range(c["axes"]):
        for j in range(c["section%d" % a]):
            i = inner + j
            freq = math.exp(-math.log(c["base"]) * (j / c["section%d" % a] if c["axis_freqs"] else i / half))
            turn = torch.polar(torch.ones(c["rows"], dtype=torch.float64, device="cuda"),
                               s["positions"][:, a].double() * (-freq if c["inverse"] else freq))
            u, w = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
            z = torch.complex(x[:, u: c["heads"] * c["head_dim"]: c["head_dim"]],
                              x[:, w: c["heads"] * c["head_dim"]: c["head_dim"]]) * turn[:, None]
            y[:, u: c["heads"] * c["head_dim"]: c["head_dim"]] = z.real
            y[:, w: c["heads"] * c["head_dim"]: c["head_dim"]] = z.imag
        inner += c["section%d" % a]
    for i in range(2 * half, c["head_dim"]):
        y[:, i: c["heads"] * c["head_dim"]: c["head_dim"]] = x[:, i: c["heads"] * c["head_dim"]: c["head_dim"]]
    return y


def _exact_store(c, s):
    width, table, off = c["kv_heads"] * c["head_dim"], s["table"].tolist(), s["offsets"].tolist()
    k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
    for b in range(c["batch"]):
        lo, hi, n = off[b], off[b + 1], c["held"]
        w[b, :, n: n + hi - lo] = 0.0
        while lo < hi:   # page by page
            at = n % c["page"]
            step = min(hi - lo, c["page"] - at)
            for pool, col in ((k, 0), (v, width)):
                part = s["rows"][lo: lo + step, col: col + width].double()
                pool[table[b][n // c["page"]], :, at: at + step] = part.view(step, c["kv_heads"], -1).transpose(0, 1)
            lo, n = lo + step, n + step
    return {"k": k, "v": v, "weights": w, "positions": None, "new_lengths": None, "new_seen": None}


def _exact_attention(c, s):
    B, H, D, group = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(B, c["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, : -(-n // c["page"])].long()
        for h in range(H):
            k = s["k"][pages, h].reshape(-1, D)[:n].double()
            v = s["v"][pages, h].reshape(-1, D)[:n].double()
            q = s["q"].view(B, c["heads"], D)[b, h * group: (h + 1) * group].double()
            z = torch.mm(q, k.t()) * D ** -0.5
            lse[b, h * group: (h + 1) * group] = torch.logsumexp(z, 1)
            p = torch.softmax(z, 1)
            out[b, h * group: (h + 1) * group] = torch.mm(p, v)
            weights[b, h, :n] += p.sum(0)
    got = {"out": out.view(B, -1), "lse": lse}
    if c["weights"]:
        got["weights"] = weights
    return got


def _exact_evict(c, s):
    k, v, w = s["k"].double(), s["v"].double(), s["new_weights"].double()
    old = s["weights"].double().cpu().numpy()
    pos, seen, table = s["positions"].cpu().numpy(), s["seen"].tolist(), s["table"].long()
    for b, n in enumerate(s["lengths"].tolist()):
        for h in range(c["kv_heads"]):
            if n <= c["budget"]:
                w[b, h, :n] = s["weights"][b, h, :n].double()
                continue
            late = pos[b, h, :n] >= seen[b] - c["recent"]
            # by lateness, then weight, then the lowest slot
            best = sorted(range(n), key=lambda i: (not late[i], 0.0 if late[i] else -old[b, h, i], i))[: c["budget"]]
            kept = set(best)
            free = [i for i in range(c["budget"]) if i not in kept]
            move = sorted(i for i in kept if i >= c["budget"])
            w[b, h, : c["budget"]] = s["weights"][b, h, : c["budget"]].double()
            if not move:
                continue
            to, at = torch.tensor(free, device="cuda"), torch.tensor(move, device="cuda")
            w[b, h, to] = s["weights"][b, h, at].double()
            for pool in (k, v):
                pool[table[b, to // c["page"]], h, to % c["page"]] = \
                    pool[table[b, at // c["page"]], h, at % c["page"]]
    return {"k": k, "v": v, "new_weights": w, "new_positions": None, "new_lengths": None}
