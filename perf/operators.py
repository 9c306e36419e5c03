"""The page and rotary operators on real work: what a decode mesh does with the keys and values that a reshard brought it.

A page cache is a set of pools (one store per layer and per keys / values, pages along dim 0, heads sharded over the
devices) and three int32 stores: table[S, B] (page ids of a sequence), lengths[S] (tokens) and refs[P] (users of a
page).  A pass is one call as a scheduler makes it.  Where a pass changes the three tables, it starts by writing the
scheduler's tables of this step into them, as one copy, so that it can be repeated; page contents need none of that, as
pages that are given out or moved to were free before.

Cases (kind: what it stands for)
  copy     pages copied one by one: a prefix kept apart from the sequence that made it
  fork     sequences that go on from a common one: samples of one prompt, beams; full pages are shared, the last,
           partly filled one is copied
  free     prompts admitted (extend) and sequences that end (free) in the same scheduler step
  compact  live pages moved to the front, the tables renamed: before a pool shrinks or is offloaded
  write    queries turned in place of a copy, keys turned and written to their pages, values written: one layer of a
           decode step (one token a sequence) or of a prefill (ragged prompts)
  rotary   rotary positions on a sharded array, forward and backward: one layer of a training step
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "s8": torch.int8}
NAMES = {"bf16": "BF16", "f16": "F16", "f32": "F32", "s8": "S8"}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "s8": 1}


def _cache(kind, dev, pools, pages, tokens, heads, dim, type, seqs, blocks, used, longest, n=0):
    """dev devices that hold `heads` heads each; `used` of the `seqs` rows hold sequences of 1..longest tokens."""
    return dict(kind=kind, dev=dev, pools=pools, pages=pages, tokens=tokens, heads=heads, dim=dim, type=type, seqs=seqs,
                blocks=blocks, used=used, longest=longest, n=n)


def _write(dev, qheads, heads, dim, rotary, interleaved, type, tokens, seqs, count, before, parts=0):
    """`seqs` sequences that hold up to `before` tokens and get `count` more in all: one each in a decode step
    (count = seqs), else ragged stretches of up to twice the mean."""
    blocks = -(-(before + 2 * (count // seqs) + 3) // tokens)
    return dict(kind="write", dev=dev, qheads=qheads, heads=heads, dim=dim, rotary=rotary, interleaved=interleaved, type=type,
                tokens=tokens, seqs=seqs, count=count, before=before, blocks=blocks, pages=seqs * blocks + 3, parts=parts)


def _rotary(dev, batch, heads, seq, dim, rotary, interleaved, type, back, seq_minor, parts, far=0):
    """dev tiles of `seq` positions of an array [batch, heads, seq * dev, dim]; far: the position of the first token."""
    return dict(kind="rotary", dev=dev, batch=batch, heads=heads, seq=seq, dim=dim, rotary=rotary, interleaved=interleaved,
                type=type, back=back, seq_minor=seq_minor, parts=parts, far=far)


def listed():
    return [
        # a prefix of 64 tokens of one layer set aside: launch latency
        dict(_cache("copy", 1, 2, 64, 16, 8, 128, "bf16", 4, 16, 2, 200, 4), name="copy_few"),
        # 512 pages of 12 pools on 4 devices: the pages of a long shared document, bandwidth
        dict(_cache("copy", 4, 12, 2048, 16, 8, 128, "bf16", 8, 256, 4, 4000, 512), name="copy_many"),
        # 4 samples of one prompt
        dict(_cache("fork", 1, 2, 512, 16, 8, 128, "bf16", 16, 64, 4, 1000, 4), name="fork_beams"),
        # 256 samples of 16 long prompts, 24 layers of keys and values, 8-bit pools
        dict(_cache("fork", 1, 48, 2500, 32, 8, 128, "s8", 300, 128, 16, 4096, 256), name="fork_many"),
        # a step that admits 6 prompts and drops them
        dict(_cache("free", 1, 1, 1024, 16, 1, 8, "s8", 32, 64, 8, 900, 6), name="free_few"),
        # a whole batch of 768 long prompts admitted and dropped; the pools are not touched
        dict(_cache("free", 1, 1, 400000, 16, 1, 8, "s8", 1024, 256, 200, 4096, 768), name="free_many"),
        # a small cache of odd pages (5 tokens, 3 heads of 20): 600 bytes a page
        dict(_cache("compact", 2, 2, 301, 5, 3, 20, "f16", 24, 60, 16, 90), name="compact_odd"),
        # a fragmented cache of 16 pools: a gigabyte to move
        dict(_cache("compact", 1, 16, 8192, 16, 16, 128, "bf16", 96, 256, 64, 2048), name="compact_many"),
        # one token of 64 sequences, 32 query heads on 8 key heads
        dict(_write(1, 32, 8, 128, 128, False, "bf16", 16, 64, 64, 2000), name="write_decode"),
        # ragged prompts, half of each row turned in pairs, on 4 devices
        dict(_write(4, 8, 2, 128, 64, True, "f16", 16, 9, 18001, 1500), name="write_prefill"),
        # odd sizes in 32 bits, 60 of 84 turned, far positions scaled by parts
        dict(_rotary(1, 3, 5, 1001, 84, 60, True, "f32", False, True, 1, 1 << 20), name="rotary_odd"),
        # the gradient of the sequence-sharded heads [4,32,2048,128], stored [b,s,h,d] on 8 devices
        dict(_rotary(8, 4, 32, 256, 128, 128, False, "bf16", True, False, 1), name="rotary_backward"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["copy", "fork", "free", "compact", "write", "rotary"])
    type = rng.choice(["bf16", "f16", "f32"])
    dim = rng.choice([16, 40, 64, 80, 96, 100, 128, 192, 256])
    if kind in ("copy", "fork", "compact"):
        tokens, heads, dev = rng.choice([1, 5, 8, 16, 32, 64]), rng.randint(1, 12), rng.choice([1, 1, 2, 4])
        type = rng.choice(["bf16", "f16", "f32", "s8"])
        pools = rng.randint(1, 16)
        page = dev * pools * tokens * heads * dim * SIZE[type]
        pages = max(48, min(_log(rng, 64, 20000), (4 << 30) // page))
        used = rng.randint(1, 12)
        longest = max(1, (pages // 2 // used - 1) * tokens - rng.randint(0, tokens - 1))
        n = max(1, min(_log(rng, 1, 1000), pages // 4))
        return _cache(kind, dev, pools, pages, tokens, heads, dim, type, used + max(n, 3), -(-longest // tokens) + 1, used, longest, n)
    if kind == "free":
        n, used, tokens = _log(rng, 1, 700), rng.randint(1, 100), rng.choice([1, 8, 16, 32])
        longest = _log(rng, 1, 8000)
        blocks = -(-longest // tokens) + 1
        while (n + used) * blocks > 400000:
            longest = max(1, longest // 2)
            blocks = -(-longest // tokens) + 1
        return _cache(kind, 1, 1, (n + used) * blocks + rng.randint(0, 500), tokens, 1, 8, "s8", n + used + 3, blocks, used, longest, n)
    rotary = 2 * rng.randint(1, dim // 2) if rng.random() < 0.3 else dim
    interleaved, parts = rng.random() < 0.5, rng.randint(0, 2)
    if kind == "write":
        heads = rng.randint(1, 8)
        seqs = _log(rng, 1, 128)
        dev = rng.choice([1, 1, 2, 4])
        room = (2 << 30) // (2 * dev * heads * dim * SIZE[type] * seqs)  # tokens a sequence may hold in 2 GiB of pools
        count = seqs if rng.random() < 0.4 else max(seqs, min(_log(rng, 1, 16000), room // 4 * seqs))
        return _write(dev, heads * rng.choice([1, 2, 4]), heads, dim, rotary, interleaved, type, rng.choice([1, 5, 16, 32, 64]),
                      seqs, count, max(1, min(_log(rng, 1, 4000), room // 2)), parts)
    return _rotary(rng.choice([1, 2, 4]), rng.randint(1, 4), rng.randint(1, 32), _log(rng, 1, 1500), dim, rotary, interleaved, type,
                   rng.random() < 0.5, rng.random() < 0.5, parts, rng.choice([0, 0, 1 << 17]))


# ---------------------------------------------------------------- inputs

def _table(c, g):
    """Sequences in a fragmented pool: page ids drawn without repetition; every second sequence shares a stretch of
    full pages with the one before it."""
    S, B, T, P, used = c["seqs"], c["blocks"], c["tokens"], c["pages"], c["used"]
    lengths = torch.zeros(S, dtype=torch.int64, device="cuda")
    lengths[:used] = torch.randint(1, c["longest"] + 1, (used,), device="cuda", generator=g)
    have = (lengths + T - 1) // T
    at = torch.arange(B, device="cuda")[None, :]
    order = torch.randperm(P, device="cuda", generator=g)
    start = torch.cumsum(have, 0) - have
    table = order[(start[:, None] + at).clamp(max=P - 1)]
    share = torch.zeros(S, dtype=torch.int64, device="cuda")
    share[1:] = torch.minimum(lengths[1:] // T, lengths[:-1] // T) // 2
    share[::2] = 0
    table = torch.where(at < share[:, None], table.roll(1, 0), table)
    live = at < have[:, None]
    refs = torch.zeros(P, dtype=torch.int64, device="cuda").scatter_add_(0, table[live], torch.ones_like(table[live]))
    return table, lengths, refs


def _frequencies(c):
    """Turns a position advances each pair by, in 64 bits, and the magnitude; parts 0: plain, 1: scaled by parts of the
    spectrum for a context 8 times longer than the 4096 tokens of training, 2: positions divided by 4."""
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / c["rotary"]) / (2.0 * math.pi)
    if c["parts"] == 1:
        w = ((4096.0 * f - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * (w + (1.0 - w) / 8.0), 1.0 + 0.1 * math.log(8.0)
    return (f / 4.0 if c["parts"] == 2 else f), 1.0


def _rotary_plan(ctx, c):
    scaling = {0: {}, 1: dict(scaling="parts", factor=8.0, original_positions=4096, low_turns=1.0, high_turns=32.0,
                              magnitude=1.0 + 0.1 * math.log(8.0)), 2: dict(scaling="linear", factor=4.0)}[c["parts"]]
    return ctx.CreateRotary(c["rotary"], base=10000.0, interleaved=c["interleaved"], **scaling)


def _buffers(lead, shape, type):
    """One buffer of `shape` for each of `lead`, every one of them at a multiple of 16 bytes, seen as one tensor."""
    n = math.prod(shape)
    return torch.empty(*lead, (n + 15) // 16 * 16, dtype=type, device="cuda")[..., :n].unflatten(-1, shape)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    type = TYPES[c["type"]]
    new = lambda *shape: _buffers(shape[:1], shape[1:], type).normal_(generator=g)  # noqa: E731
    s = {"c": c}
    if c["kind"] == "rotary":
        shape = (c["dev"], c["batch"], c["heads"], c["seq"], c["dim"]) if c["seq_minor"] else (c["dev"], c["batch"], c["seq"], c["heads"], c["dim"])
        s["x"], s["out"] = new(*shape), _buffers(shape[:1], shape[1:], type)
    elif c["kind"] == "write":
        before = torch.randint(0, c["before"] + 1, (c["seqs"],), device="cuda", generator=g)
        n, share = c["count"], c["count"] // c["seqs"]
        begins = torch.arange(c["seqs"] + 1, device="cuda") * n // c["seqs"]
        if share > 1:
            begins[1:-1] += torch.randint(-(share // 2), share // 2 + 1, (c["seqs"] - 1,), device="cuda", generator=g)
        count = begins[1:] - begins[:-1]
        s["table"] = torch.randperm(c["pages"], device="cuda", generator=g)[:c["seqs"] * c["blocks"]].view(c["seqs"], c["blocks"]).int()
        s["lengths"], s["begins"] = (before + count).int(), begins.int()
        s["refs"] = torch.ones(c["pages"], dtype=torch.int32, device="cuda")
        s["slots"] = torch.randperm(c["seqs"], device="cuda", generator=g).int()
        s["lengths"] = torch.empty_like(s["lengths"]).index_copy_(0, s["slots"].long(), s["lengths"])
        s["q"], s["k"], s["v"] = new(c["dev"], n, c["qheads"], c["dim"]), new(c["dev"], n, c["heads"], c["dim"]), new(c["dev"], n, c["heads"], c["dim"])
        s["q_out"] = _buffers(s["q"].shape[:1], s["q"].shape[1:], type)
        s["pools"] = _buffers((2, c["dev"]), (c["pages"], c["tokens"], c["heads"], c["dim"]), type).normal_(generator=g)
    else:
        pools = s["pools"] = _buffers((c["pools"], c["dev"]), (c["pages"], c["tokens"], c["heads"], c["dim"]), type)
        pools.random_(-127, 128, generator=g) if c["type"] == "s8" else pools.normal_(generator=g)
        table, lengths, refs = _table(c, g)
        # one buffer, each part at a multiple of 4 values: a scheduler sends its tables in one copy
        sizes = [(t.numel() + 3) // 4 * 4 for t in (table, lengths, refs)]
        s["step"] = torch.cat([torch.nn.functional.pad(t.flatten(), (0, m - t.numel())) for t, m in zip((table, lengths, refs), sizes)]).int()
        s["now"] = s["step"].clone()
        parts = s["now"].split(sizes)
        s["table"], s["lengths"], s["refs"] = (p[:t.numel()].view(t.shape) for p, t in zip(parts, (table, lengths, refs)))
        s["n"] = c["n"]
        if c["kind"] == "copy":
            pick = torch.randperm(c["pages"], device="cuda", generator=g)[:2 * c["n"]].int()
            s["src"], s["dst"] = pick[:c["n"]].contiguous(), pick[c["n"]:].contiguous()
        elif c["kind"] == "fork":
            s["parents"] = torch.randint(0, c["used"], (c["n"],), device="cuda", generator=g).int()
            s["children"] = (torch.randperm(c["seqs"] - c["used"], device="cuda", generator=g)[:c["n"]] + c["used"]).int()
        elif c["kind"] == "free":
            s["slots"] = (torch.randperm(c["seqs"] - c["used"], device="cuda", generator=g)[:c["n"]] + c["used"]).int()
            s["counts"] = torch.randint(1, c["longest"] + 1, (c["n"],), device="cuda", generator=g).int()
    if own:
        _handles(s, c)
    return s


def _handles(s, c):
    """What a program keeps beside its buffers: the context on its stream, the stores, the cache and the rotary plan."""
    import multimesh_jax_amd as mm
    s["stream"] = torch.cuda.Stream()
    ctx = s["ctx"] = mm.ReshardContext(0, hip_stream=s["stream"].cuda_stream)
    name, dev = NAMES[c["type"]], c["dev"]

    def store(t, type, shape, cut=None):
        """t[k] is the buffer of device k; dim `cut` is sharded over the devices."""
        dims = [(n * (dev if i == cut else 1), dev if i == cut else 1, i) for i, n in enumerate(shape)]
        devices = 1 if cut is None else dev
        return ctx.AdoptShards(mm.sharded_shape(type, dims, 0, devices), [t[k].data_ptr() for k in range(devices)])

    if c["kind"] == "rotary":
        shape = s["x"].shape[1:]
        at = 2 if c["seq_minor"] else 1
        s["plan"], s["at"] = _rotary_plan(ctx, c), at
        s["x_store"], s["out_store"] = store(s["x"], name, shape, at), store(s["out"], name, shape, at)
        return
    if c["kind"] == "write":
        s["plan"] = _rotary_plan(ctx, c)
        for part in ("q", "k", "v", "q_out"):
            s[part + "_store"] = store(s[part], name, s[part].shape[1:], 1)
    pools = [store(p, name, p.shape[1:], 2) for p in s["pools"]]
    tables = [store(t[None], "S32", t.shape) for t in (s["table"], s["lengths"], s["refs"])]
    s["cache"] = ctx.CreatePages(pools, *tables, page_tokens=c["tokens"])


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["c"]
    if own:
        return _own(s, c)
    return {"copy": _copy, "fork": _fork, "free": _free, "compact": _compact, "write": _plain_write, "rotary": _plain_rotary}[c["kind"]](s, c)


def _own(s, c):
    kind = c["kind"]
    if kind == "rotary":
        s["ctx"].ApplyRotary(s["plan"], s["x_store"], s["out_store"], seq_dim=s["at"], offset=c["far"], backward=c["back"])
        return s["out"]
    cache = s["cache"]
    if kind == "write":
        cache.Write(s["slots"], s["begins"], 0, s["k_store"], 1, s["v_store"], rotary=s["plan"], q=s["q_store"], q_out=s["q_out_store"])
        return s["q_out"], s["pools"]
    if kind == "copy":
        cache.Copy(s["src"], s["dst"])
        return s["pools"]
    with torch.cuda.stream(s["stream"]):
        s["now"].copy_(s["step"])
    if kind == "fork":
        cache.Fork(s["parents"], s["children"])
        return s["pools"], s["now"]
    if kind == "free":
        cache.Extend(s["slots"], s["counts"])
        cache.Free(s["slots"])
        return s["now"]
    cache.Compact()
    return s["pools"], s["now"]


# ---------------------------------------------------------------- plain forms

def _copy(s, c):
    s["pools"].index_copy_(2, s["dst"].long(), s["pools"].index_select(2, s["src"].long()))
    return s["pools"]


def _lowest_free(refs):
    """ids[k] = the k-th free page."""
    P = refs.numel()
    free = refs == 0
    at = torch.where(free, torch.cumsum(free, 0) - 1, P)
    return torch.empty(P + 1, dtype=torch.int64, device=refs.device).scatter_(0, at, torch.arange(P, device=refs.device))


def _fork(s, c):
    s["now"].copy_(s["step"])
    table, lengths, refs, T = s["table"], s["lengths"], s["refs"], c["tokens"]
    parents, children = s["parents"].long(), s["children"].long()
    l = lengths[parents]
    full, rest = (l // T).long(), l % T > 0
    fresh = _lowest_free(refs)[torch.cumsum(rest, 0) - 1]
    rows = table[parents]
    at = torch.arange(c["blocks"], device=rows.device)[None, :]
    shared = at < full[:, None]
    refs.scatter_add_(0, rows.flatten().long(), shared.flatten().int())
    last = (at == full[:, None]) & rest[:, None]
    source = rows.gather(1, full.clamp(max=c["blocks"] - 1)[:, None])[:, 0]
    table[children] = torch.where(shared, rows, torch.where(last, fresh[:, None].int(), table[children]))
    lengths[children] = l
    refs.index_put_((fresh[rest],), torch.ones_like(refs[:1]))
    s["pools"].index_copy_(2, fresh[rest], s["pools"].index_select(2, source[rest]))
    return s["pools"], s["now"]


def _free(s, c):
    s["now"].copy_(s["step"])
    table, lengths, refs, T = s["table"], s["lengths"], s["refs"], c["tokens"]
    slots, counts = s["slots"].long(), s["counts"].long()
    at = torch.arange(c["blocks"], device=refs.device)[None, :]
    old = lengths[slots]
    have, want = (old + T - 1) // T, (old + counts + T - 1) // T
    first = torch.cumsum(want - have, 0) - (want - have)
    fresh = (at >= have[:, None]) & (at < want[:, None])
    ids = _lowest_free(refs)[(first[:, None] + at - have[:, None]).clamp(0, refs.numel())]
    rows = torch.where(fresh, ids.int(), table[slots])
    table[slots] = rows
    refs.scatter_add_(0, rows[fresh].long(), torch.ones_like(rows[fresh]))
    lengths[slots] = (old + counts).int()
    # the same sequences end
    rows, live = table[slots], at < (lengths[slots] + T - 1)[:, None] // T
    refs.scatter_add_(0, rows[live].long(), torch.full_like(rows[live], -1))
    lengths[slots] = 0
    return s["now"]


def _compact(s, c):
    s["now"].copy_(s["step"])
    table, lengths, refs, T = s["table"], s["lengths"], s["refs"], c["tokens"]
    ids = torch.arange(c["pages"], device=refs.device)
    live = refs > 0
    count = live.sum()
    src, dst = ids[live & (ids >= count)], ids[~live & (ids < count)]
    s["pools"].index_copy_(2, dst, s["pools"].index_select(2, src))
    name = ids.index_copy(0, src, dst)
    held = torch.arange(c["blocks"], device=refs.device)[None, :] < ((lengths + T - 1) // T)[:, None]
    table.copy_(torch.where(held, name[table.long()].int(), table))
    refs.index_copy_(0, dst, refs[src])
    refs.index_fill_(0, src, 0)
    return s["pools"], s["now"]


def _turn(x, positions, c, back):
    """x[..., dim] in 32 bits, positions broadcast over x's leading dims."""
    R = c["rotary"]
    f, magnitude = _frequencies(c)
    t = positions.double()[..., None] * f.to(x.device)
    angle = (t - t.floor()) * (2.0 * math.pi)
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * (-magnitude if back else magnitude)).float()
    x = x.float()
    turned, rest = x[..., :R], x[..., R:]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


def _positions(c, device):
    """[dev, 1, seq, 1] or its seq-minor form: where each row of the array stands."""
    p = c["far"] + torch.arange(c["dev"] * c["seq"], device=device).view(c["dev"], 1, 1, c["seq"])
    return p if c["seq_minor"] else p.transpose(2, 3)


def _plain_rotary(s, c):
    x = s["x"]
    return _turn(x, _positions(c, x.device), c, c["back"]).to(x.dtype)


def _places(s, c):
    """Position, page and row in the page of every new token."""
    begins, slots, lengths = s["begins"].long(), s["slots"].long(), s["lengths"].long()
    n = s["q"].shape[1]
    token = torch.arange(n, device=begins.device)
    j = torch.searchsorted(begins[1:], token, right=True)
    position = lengths[slots[j]] - begins[j + 1] + token
    return position, s["table"][slots[j], position // c["tokens"]].long(), position % c["tokens"]


def _plain_write(s, c):
    position, page, row = _places(s, c)
    where = position[None, :, None]
    q = _turn(s["q"], where, c, False).to(s["q"].dtype)
    k = _turn(s["k"], where, c, False).to(s["k"].dtype)
    s["pools"][0][:, page, row] = k
    s["pools"][1][:, page, row] = s["v"]
    return q, s["pools"]


# ---------------------------------------------------------------- what a pass cannot do without

def work(c):
    if c["kind"] == "rotary":
        n = c["dev"] * c["batch"] * c["heads"] * c["seq"]
        return {"bytes": 2 * n * c["dim"] * SIZE[c["type"]], "flops": 3 * n * c["rotary"]}
    if c["kind"] == "write":
        tokens = c["count"] * c["dev"]
        return {"bytes": 2 * tokens * (c["qheads"] + 2 * c["heads"]) * c["dim"] * SIZE[c["type"]],
                "flops": 3 * tokens * (c["qheads"] + c["heads"]) * c["rotary"]}
    page = c["tokens"] * c["heads"] * c["dim"] * SIZE[c["type"]] * c["pools"] * c["dev"]
    tables = 4 * (c["seqs"] * c["blocks"] + c["seqs"] + c["pages"])
    live = c["used"] * (c["longest"] + 1) / 2 / c["tokens"] * 0.88  # pages; an eighth of them shared
    rows = c["n"] * (c["longest"] + 1) / 2 / c["tokens"]
    if c["kind"] == "copy":
        return {"bytes": 2 * c["n"] * page, "flops": 0}
    if c["kind"] == "fork":
        return {"bytes": 2 * tables + 2 * c["n"] * page * (1 - 1 / c["tokens"]) + 4 * 4 * rows, "flops": 0}
    if c["kind"] == "free":
        return {"bytes": 2 * tables + 4 * c["pages"] + 4 * 6 * rows, "flops": 0}
    moved = live * max(0.0, 1 - live / c["pages"])
    return {"bytes": 2 * tables + 2 * moved * page + 4 * c["pages"] + 8 * live, "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(c, seed):
    if c["kind"] not in ("rotary", "write"):
        return None  # whole numbers and pages that move as they are
    s = prepare(c, seed)
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64, device="cuda")
    theta = torch.exp(-(2.0 * i / c["rotary"]) * math.log(10000.0))
    m = 1.0
    if c["parts"] == 1:
        keep = torch.clip((4096.0 * theta / (2.0 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        theta, m = keep * theta + (1.0 - keep) * theta / 8.0, 1.0 + 0.1 * math.log(8.0)
    elif c["parts"] == 2:
        theta = theta / 4.0

    def turned(x, p, sign):
        z = torch.polar(torch.full_like(p[..., None] * theta, m), sign * p[..., None] * theta)  # m exp(+-i p theta)
        y = x.double()
        if c["interleaved"]:
            pairs = y[..., :c["rotary"]].unflatten(-1, (-1, 2))
        else:
            pairs = y[..., :c["rotary"]].unflatten(-1, (2, -1)).transpose(-1, -2)
        v = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        y[..., :c["rotary"]] = v.flatten(-2) if c["interleaved"] else v.transpose(-1, -2).flatten(-2)
        return y

    if c["kind"] == "rotary":
        p = torch.arange(c["far"], c["far"] + c["dev"] * c["seq"], dtype=torch.float64, device="cuda").view(c["dev"], c["seq"])
        p = p[:, None, None, :] if c["seq_minor"] else p[:, None, :, None]
        return turned(s["x"], p, -1.0 if c["back"] else 1.0)
    count = (s["begins"][1:] - s["begins"][:-1]).long()
    j = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), count)
    slot = s["slots"].long()[j]
    p = s["lengths"].long()[slot] - s["begins"].long()[1:][j] + torch.arange(j.numel(), device="cuda")
    page = s["table"].long()[slot, torch.div(p, c["tokens"], rounding_mode="floor")]
    pools = s["pools"].double()
    place = (slice(None), page, p - torch.div(p, c["tokens"], rounding_mode="floor") * c["tokens"])
    pools[0][place] = turned(s["k"], p.double()[None, :, None], 1.0)
    pools[1][place] = s["v"].double()
    return turned(s["q"], p.double()[None, :, None], 1.0), pools
