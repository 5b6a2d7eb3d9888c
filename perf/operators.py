"""The paged KV cache operators, as cases that can be timed and compared.

Four operators on a cache whose slots live in pages: appending rows, the model's fused q/k norm + rope + append, decode
attention of one new token per lane (with the accumulated attention weight of every slot, the "mass"), and eviction by that mass.
``run`` computes them as plain torch, or through ``tatara_b200.Context`` where ``own`` is true.

A cache here is a pair of pools viewed as [page][kv head][slot][dim], a page table [lane][page of the lane] (entry -1: no page
yet), and two per-lane planes [lane][kv head][slot]: the mass (f32) and the position (i32) of the token in the slot.  ``lanes`` is
[lane][2] i32: slots in use, the newest token's included (0: an idle lane), and the newest token's position.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_PAIRS, ROPE_BASE, RMS_EPS = 32, 1.0e7, 1e-6
MODEL = {"dtype": "bf16", "q_heads": 16, "kv_heads": 2, "dim": 256}   # the gated attention layers of this framework


# ---- cases -------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # One conversation of about a thousand tokens: two short launches, latency is all of it.
        {"name": "decode 1 lane 1000", "op": "decode", **MODEL, "page": 16, "slot_major": False, "lanes": 1, "shortest": 1000,
         "longest": 1000, "idle": False, "gate": True, "mass": False},
        # The model's longest context on one lane: the whole card streams one cache.
        {"name": "decode 1 lane 262144", "op": "decode", **MODEL, "page": 64, "slot_major": False, "lanes": 1, "shortest": 262144,
         "longest": 262144, "idle": False, "gate": True, "mass": False},
        # A serving batch of 32 lanes whose caches are trimmed: the mass is kept up at every token.
        {"name": "decode 32 lanes mass", "op": "decode", **MODEL, "page": 64, "slot_major": False, "lanes": 32, "shortest": 4096,
         "longest": 32768, "idle": False, "gate": True, "mass": True},
        # Another head layout (32 query and 8 kv heads of 128, half precision, slot-major pages), odd lengths and a padded lane.
        {"name": "decode 7 lanes f16 d128", "op": "decode", "dtype": "f16", "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "slot_major": True, "lanes": 7, "shortest": 17, "longest": 5003, "idle": True, "gate": False, "mass": True},
        # Many short lanes of a small model without shared heads.
        {"name": "decode 96 lanes d64", "op": "decode", "dtype": "bf16", "q_heads": 12, "kv_heads": 12, "dim": 64, "page": 32,
         "slot_major": True, "lanes": 96, "shortest": 40, "longest": 1500, "idle": False, "gate": False, "mass": False},
        # One new row for each of eight lanes: the least an append can be.
        {"name": "append 8 lanes 1 row", "op": "append", "dtype": "f16", "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "slot_major": True, "lanes": 8, "shortest": 100, "longest": 4000, "rows": 1},
        # Prompts of four lanes, prefilled in a contiguous lane cache, taken over into pages.
        {"name": "append 4 prompts 30001", "op": "append", **MODEL, "page": 64, "slot_major": False, "lanes": 4, "shortest": 9000,
         "longest": 30001, "rows": 0},
        # A decode token of eight lanes through the model's own projection row.
        {"name": "rope 8 lanes", "op": "rope", **MODEL, "page": 16, "slot_major": False, "lanes": 8, "shortest": 300,
         "longest": 9000, "history": 0},
        # The largest batch, its caches trimmed: few slots, positions close to the model's longest context.
        {"name": "rope 256 lanes", "op": "rope", **MODEL, "page": 16, "slot_major": False, "lanes": 256, "shortest": 20,
         "longest": 600, "history": 250000},
        # A lane of 4096 slots that has decoded 100 tokens more and is trimmed back.
        {"name": "evict 1 lane 4196", "op": "evict", **MODEL, "page": 16, "slot_major": False, "lanes": 1, "shortest": 4196,
         "longest": 4196, "keep": 4096, "sink": 4, "recent": 512, "history": 20000},
        # A ragged batch trimmed to a quarter of its longest lane; the shorter lanes stay as they are.
        {"name": "evict 24 lanes f16", "op": "evict", "dtype": "f16", "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "slot_major": True, "lanes": 24, "shortest": 2500, "longest": 16000, "keep": 4000, "sink": 16, "recent": 999, "history": 0},
        # A prompt at the model's longest context cut to a quarter.
        {"name": "evict 1 lane 262144", "op": "evict", **MODEL, "page": 64, "slot_major": False, "lanes": 1, "shortest": 262144,
         "longest": 262144, "keep": 65536, "sink": 64, "recent": 8192, "history": 0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A case of the listed ranges: any head layout the operators take, one lane to many, one token to the longest lane."""
    op = rng.choice(["decode", "decode", "decode", "append", "rope", "evict", "evict"])
    layout = dict(MODEL)
    if op != "rope" and rng.random() < 0.6:
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        layout = {"dtype": rng.choice(["bf16", "f16"]), "q_heads": kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16]),
                  "kv_heads": kv_heads, "dim": dim}
    case = {"op": op, **layout, "page": rng.choice([16, 32, 48, 64, 128]), "slot_major": op != "rope" and rng.random() < 0.5}
    row = 4 * layout["kv_heads"] * layout["dim"]                  # bytes of a slot, K and V
    if op == "rope":
        case["lanes"] = _spread(rng, 1, 256)
        case["longest"] = _spread(rng, 1, 2000)
        case["history"] = rng.choice([0, 1000, 120000])
    else:
        case["lanes"] = _spread(rng, 1, 64)
        most = min(200000, 300_000_000 // row) // case["lanes"]   # slots of all lanes: 300 MB
        case["longest"] = _spread(rng, 64 if op == "evict" else 1, max(128, most))
    case["shortest"] = max(1, int(case["longest"] * rng.choice([1.0, 0.6, 0.2, 0.05])))
    if op == "decode":
        case.update(idle=rng.random() < 0.3, gate=rng.random() < 0.5, mass=rng.random() < 0.5)
    elif op == "append":
        case["rows"] = rng.choice([0, 0, 1, 3])
    elif op == "evict":
        case["keep"] = max(8, int(case["longest"] * rng.uniform(0.1, 0.95)))
        case["sink"] = rng.randint(0, case["keep"] // 8)
        case["recent"] = rng.randint(0, case["keep"] // 4)
        case["history"] = rng.choice([0, 0, 777])
    return case


def _lengths(case):
    """Slots in use of every lane: the longest first, the others spread over the logarithm; an idle lane comes last."""
    rng = random.Random(case["lanes"] * 1000003 + case["longest"])
    got = [case["longest"]] + [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["lanes"] - 1)]
    if case.get("idle") and case["lanes"] > 1:
        got[-1] = 0
    return got


def _appended(case):
    """Rows that an append brings for every lane: `rows` newest ones, or with 0 the whole lane."""
    return [min(n, case["rows"]) if case["rows"] else n for n in _lengths(case)]


# ---- inputs ------------------------------------------------------------------------------------------------------------


def _cache(case, lens, gen, history=0):
    """Pools with the lanes' pages in random order, some pages to spare, and not-a-number wherever no token was written."""
    page, heads, dim, dtype = case["page"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    per_lane = [-(-n // page) for n in lens]
    columns = max(per_lane) + 2
    pages = sum(per_lane) + 5
    order = torch.randperm(pages, generator=gen, device=DEVICE, dtype=torch.int32)
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device=DEVICE)
    shape = (pages, page, heads, dim) if case["slot_major"] else (pages, heads, page, dim)
    pools, at = [], 0
    for _ in range(2):
        pool = torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)
        pools.append(pool.permute(0, 2, 1, 3) if case["slot_major"] else pool)
    for lane, n in enumerate(lens):
        table[lane, : per_lane[lane]] = order[at: at + per_lane[lane]]
        at += per_lane[lane]
        if n % page:
            for pool in pools:
                pool[int(table[lane, per_lane[lane] - 1]), :, n % page:] = float("nan")
    for pool in pools:
        pool[order[at:].long()] = float("nan")
    lanes = torch.tensor([[n, max(0, history + n - 1)] for n in lens], dtype=torch.int32, device=DEVICE)
    return {"keys": pools[0], "values": pools[1], "table": table, "lanes": lanes, "page": page}


def _planes(case, lens, columns, gen, history):
    """[2][lane][kv head][slot] i32: the masses (their bits), then the positions."""
    slots = columns * case["page"]
    planes = torch.zeros((2, len(lens), case["kv_heads"], slots), dtype=torch.int32, device=DEVICE)
    mass = planes[0].view(torch.float32)
    # attention weight is spread unevenly: most slots have got little, the first ones of a lane much
    mass.copy_(torch.exp(2.0 * torch.randn(mass.shape, generator=gen, device=DEVICE) - 3.0))
    mass[:, :, :4] += 50.0
    mass[:, :, 5::97] = 0.0        # slots that no query has looked at yet
    planes[1] = torch.arange(slots, dtype=torch.int32, device=DEVICE)
    if history:
        for lane, n in enumerate(lens):   # trimmed before: the kept slots hold a scattered choice of the older positions
            first = min(case["sink"], n)
            old = max(first, min(n, case["keep"]) - case["recent"] // 2)
            for head in range(case["kv_heads"]):
                seen = torch.randperm(history + old - first, generator=gen, device=DEVICE)[: old - first]
                planes[1, lane, head, first:old] = seen.to(torch.int32) + first
            planes[1, lane, :, old:n] = torch.arange(history + old, history + n, dtype=torch.int32, device=DEVICE)
    return planes


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) & 0x7FFFFFFF)
    lens = _lengths(case)
    dtype, heads, dim = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    state = {"op": case["op"], "longest": max(lens), **_cache(case, lens, gen, case.get("history", 0))}
    columns = state["table"].shape[1]
    if case["op"] == "decode":
        shape = (case["lanes"], case["q_heads"], dim)
        # heads differ in how sharply they look: temperatures from 0.5 to 3
        warmth = 0.5 + 2.5 * torch.rand((1, case["q_heads"], 1), generator=gen, device=DEVICE)
        state["q"] = (torch.randn(shape, generator=gen, device=DEVICE) * warmth).to(dtype)
        state["gate"] = torch.randn(shape, generator=gen, device=DEVICE).to(dtype) if case["gate"] else None
        state["out"] = torch.zeros(shape, dtype=dtype, device=DEVICE)
        state["scale"] = dim ** -0.5
        state["mass"] = None
        if case["mass"]:
            state["mass"] = torch.rand((case["lanes"], heads, columns * case["page"]), generator=gen, device=DEVICE)
    elif case["op"] == "append":
        counts = _appended(case)
        starts = np.concatenate([[0], np.cumsum(counts)])
        rows = int(starts[-1])
        state["row_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        if case["slot_major"]:
            source = [torch.randn((rows, heads, dim), generator=gen, device=DEVICE, dtype=dtype) for _ in range(2)]
        else:   # the planes of a contiguous cache, [kv head][row][dim], with room behind the rows
            source = [torch.randn((heads, rows + 64, dim), generator=gen, device=DEVICE, dtype=dtype)[:, :rows].transpose(0, 1) for _ in range(2)]
        state["new_keys"], state["new_values"] = source
        planes = torch.zeros((2, case["lanes"], heads, columns * case["page"]), dtype=torch.int32, device=DEVICE)
        state["mass"], state["positions"] = planes[0].view(torch.float32), planes[1]
        state["mass"].fill_(1.0)
    elif case["op"] == "rope":
        lanes = case["lanes"]
        state["projection"] = torch.randn((lanes, 9216), generator=gen, device=DEVICE).to(dtype)
        for name in ("q_weight", "k_weight"):
            state[name] = (1.0 + 0.1 * torch.randn(dim, generator=gen, device=DEVICE)).to(dtype)
        state["q"], state["gate"] = (torch.zeros((lanes, 16, dim), dtype=dtype, device=DEVICE) for _ in range(2))
        state["divisors"] = torch.tensor(_divisors(), device=DEVICE)
        planes = torch.zeros((2, lanes, heads, columns * case["page"]), dtype=torch.int32, device=DEVICE)
        state["mass"], state["positions"] = planes[0].view(torch.float32), planes[1]
        state["mass"].fill_(1.0)
    else:
        # a pass trims the same cache again: the planes are put back first (K and V of the slots that move stay behind as they were)
        state["before"] = _planes(case, lens, columns, gen, case["history"])
        state["planes"] = state["before"].clone()
        state["mass"], state["positions"] = state["planes"][0].view(torch.float32), state["planes"][1]
        state.update(keep=case["keep"], sink=case["sink"], recent=case["recent"])
    if own:
        _handles(state, case)
    return state


def _divisors():
    return np.power(ROPE_BASE, np.arange(ROPE_PAIRS) / ROPE_PAIRS).astype(np.float32)


_context = None


def _handles(state, case):
    """What a program that serves from this cache keeps: the context, the cache's descriptor and the scratch."""
    global _context
    import tatara_b200 as tb
    if _context is None:
        _context = tb.Context(torch.cuda.current_device())
    state["ctx"] = _context
    state["cache"] = tb.paged_cache(state["keys"], state["values"], state["table"], mass=state.get("mass"), positions=state.get("positions"))
    if case["op"] == "decode":
        need = tb.decode_paged_scratch_bytes(state["cache"], case["lanes"], state["longest"], case["q_heads"])
        state["scratch"] = torch.empty(need, dtype=torch.uint8, device=DEVICE)
    elif case["op"] == "evict":
        need = tb.paged_evict_scratch_bytes(state["cache"], case["lanes"], state["longest"], case["keep"])
        state["scratch"] = torch.empty(need, dtype=torch.uint8, device=DEVICE)


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _gathered(pool, table, live):
    """[lane][kv head][slot][dim] in 32 bits out of the pages; nothing where a slot is not in use."""
    got = pool[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)
    got = got.reshape(got.shape[0], got.shape[1], -1, got.shape[-1]).float()
    return torch.where(live[:, None, :, None], got, 0.0)


def _decode(s):
    table = s["table"][:, : -(-s["longest"] // s["page"])]
    slots = table.shape[1] * s["page"]
    live = torch.arange(slots, device=DEVICE)[None, :] < s["lanes"][:, :1]
    q = s["q"].float()
    lanes, q_heads, dim = q.shape
    heads = s["keys"].shape[1]
    scores = q.view(lanes, heads, q_heads // heads, dim) @ _gathered(s["keys"], table, live).transpose(2, 3) * s["scale"]
    scores = torch.where(live[:, None, None, :], scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(dim=-1, keepdim=True)
    weights = weights / torch.where(total == 0.0, 1.0, total)
    out = (weights @ _gathered(s["values"], table, live)).reshape(lanes, q_heads, dim)
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    s["out"].copy_(out)
    if s["mass"] is not None:
        s["mass"][:, :, :slots] += weights.sum(dim=2)


def _write_rows(s, lane, slot, position, keys, values):
    page, row = s["table"][lane, slot // s["page"]].long(), slot % s["page"]
    s["keys"].permute(0, 2, 1, 3)[page, row] = keys
    s["values"].permute(0, 2, 1, 3)[page, row] = values
    s["mass"].permute(0, 2, 1)[lane, slot] = 0.0
    s["positions"].permute(0, 2, 1)[lane, slot] = position[:, None].to(torch.int32)


def _append(s):
    starts = s["row_starts"].long()
    row = torch.arange(s["new_keys"].shape[0], device=DEVICE)
    lane = torch.searchsorted(starts, row, right=True) - 1
    back = starts[lane + 1] - row            # 1 for a lane's newest row
    held = s["lanes"].long()[lane]
    _write_rows(s, lane, held[:, 0] - back, held[:, 1] + 1 - back, s["new_keys"], s["new_values"])


def _normed(x, weight):
    x = x.float()
    return weight.float() * (x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + RMS_EPS))


def _rotated(x, sine, cosine):
    low, high = x[..., :ROPE_PAIRS], x[..., ROPE_PAIRS: 2 * ROPE_PAIRS]
    return torch.cat([low * cosine - high * sine, high * cosine + low * sine, x[..., 2 * ROPE_PAIRS:]], dim=-1)


def _rope(s):
    rows = s["projection"].shape[0]
    position = s["lanes"][:, 1]
    angle = position.double()[:, None] / s["divisors"].double()      # far positions lose their angle in 32 bits
    sine, cosine = torch.sin(angle).float()[:, None, :], torch.cos(angle).float()[:, None, :]
    pairs = s["projection"][:, :8192].view(rows, 16, 2, 256)
    s["q"].copy_(_rotated(_normed(pairs[:, :, 0], s["q_weight"]), sine, cosine))
    s["gate"].copy_(pairs[:, :, 1])
    keys = _rotated(_normed(s["projection"][:, 8192:8704].view(rows, 2, 256), s["k_weight"]), sine, cosine)
    lane = torch.arange(rows, device=DEVICE)
    _write_rows(s, lane, s["lanes"][:, 0].long() - 1, position, keys.to(s["keys"].dtype), s["projection"][:, 8704:].view(rows, 2, 256))


def _evict(s):
    lanes, heads, columns = s["mass"].shape
    slot = torch.arange(columns, device=DEVICE)
    held = s["lanes"][:, :1, None]
    live = slot < held
    guarded = (slot < s["sink"]) | (s["positions"] + s["recent"] > s["lanes"][:, 1:, None])
    rank = torch.where(guarded, math.inf, s["mass"].nan_to_num(nan=-1.0, posinf=3.0e38))
    order = torch.sort(torch.where(live, rank, -math.inf), dim=-1, descending=True, stable=True).indices
    kept = torch.zeros((lanes, heads, columns), dtype=torch.bool, device=DEVICE)
    kept.scatter_(2, order[:, :, : s["keep"]], True)
    trimmed = held > s["keep"]
    hole = trimmed & ~kept & (slot < s["keep"])
    donor = trimmed & kept & live & (slot >= s["keep"])
    lane, head, to = hole.nonzero(as_tuple=True)          # both lists ascend: the j-th hole of a head takes its j-th donor
    origin = donor.nonzero(as_tuple=True)[2]
    page_to, page_from = (s["table"][lane, x // s["page"]].long() for x in (to, origin))
    for pool in (s["keys"], s["values"]):
        pool[page_to, head, to % s["page"]] = pool[page_from, head, origin % s["page"]]
    for plane in (s["mass"], s["positions"]):
        plane[lane, head, to] = plane[lane, head, origin]


def run(state):
    s, op = state, state["op"]
    if op == "evict":
        s["planes"].copy_(s["before"])
    if own:
        ctx, cache = s["ctx"], s["cache"]
        if op == "decode":
            ctx.attn_decode_paged(cache, s["lanes"], s["q"], s["gate"], s["out"], s["scratch"], max_keys=s["longest"], scale=s["scale"])
        elif op == "append":
            ctx.paged_append(cache, s["lanes"], s["new_keys"], s["new_values"], row_starts=s["row_starts"])
        elif op == "rope":
            ctx.attn_qk_rope_paged(cache, s["lanes"], s["projection"], s["q_weight"], s["k_weight"], s["q"], s["gate"])
        else:
            ctx.paged_evict(cache, s["lanes"], s["keep"], s["scratch"], sink=s["sink"], recent=s["recent"], max_keys=s["longest"])
    else:
        {"decode": _decode, "append": _append, "rope": _rope, "evict": _evict}[op](s)
    if op == "decode":
        return {"out": s["out"]} if s["mass"] is None else {"out": s["out"], "mass": s["mass"]}
    got = {"keys": s["keys"], "values": s["values"], "mass": s["mass"], "positions": s["positions"]}
    return {**got, "q": s["q"], "gate": s["gate"]} if op == "rope" else got


def work(case):
    lens = _lengths(case)
    total = sum(lens)
    heads, dim = case["kv_heads"], case["dim"]
    row = 4 * dim                                          # bytes of a slot of one kv head, K and V
    if case["op"] == "decode":
        bytes_ = total * heads * (row + (8 if case["mass"] else 0)) + case["lanes"] * case["q_heads"] * dim * (6 if case["gate"] else 4)
        return {"bytes": bytes_, "flops": 4 * total * case["q_heads"] * dim}
    if case["op"] == "append":
        return {"bytes": sum(_appended(case)) * heads * (2 * row + 8), "flops": 0}
    if case["op"] == "rope":
        return {"bytes": case["lanes"] * 2 * (9216 + 8192 + 1024) + 1024, "flops": case["lanes"] * 18 * 256 * 6}
    bytes_ = 0
    for n in lens:
        if n > case["keep"]:
            fresh = min(case["recent"], n - case["keep"])
            among = n - case["sink"] - case["recent"]
            moved = fresh + (case["keep"] - case["sink"] - case["recent"]) * max(0, n - case["keep"] - case["recent"]) / max(1, among)
            bytes_ += heads * (n * (8 if case["recent"] else 4) + moved * (2 * row + 16))
    return {"bytes": max(1, bytes_), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _lane_rows(pool, table, lane, head, n, page):
    slots = torch.arange(n, device=DEVICE)
    return pool[table[lane, slots // page].long(), head, slots % page]


def _exact_decode(s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    mass = None if s["mass"] is None else s["mass"].double()
    heads = s["keys"].shape[1]
    group = s["q"].shape[1] // heads
    for lane, (n, _) in enumerate(s["lanes"].tolist()):
        for head in range(heads if n else 0):
            k, v = (_lane_rows(s[x], s["table"], lane, head, n, s["page"]).double() for x in ("keys", "values"))
            of = slice(head * group, (head + 1) * group)
            p = torch.softmax(s["q"][lane, of].double() @ k.T * s["scale"], dim=-1)
            out[lane, of] = p @ v
            if s["gate"] is not None:
                out[lane, of] *= torch.sigmoid(s["gate"][lane, of].double())
            if mass is not None:
                mass[lane, head, :n] += p.sum(dim=0)
    return {"out": out} if mass is None else {"out": out, "mass": mass}


def _exact_rope(s):
    rows = s["projection"].double()
    angle = s["lanes"][:, 1].double()[:, None] / torch.tensor(_divisors(), device=DEVICE).double()
    turn = torch.polar(torch.ones_like(angle), angle)

    def head_of(x, weight):
        x = weight.double() * x * torch.rsqrt((x ** 2).sum(dim=-1, keepdim=True) / 256 + RMS_EPS)
        z = torch.complex(x[:, :ROPE_PAIRS], x[:, ROPE_PAIRS: 2 * ROPE_PAIRS]) * turn
        return torch.cat([z.real, z.imag, x[:, 2 * ROPE_PAIRS:]], dim=-1)

    q = torch.stack([head_of(rows[:, 512 * h: 512 * h + 256], s["q_weight"]) for h in range(16)], dim=1)
    # the pools hold values of their type: what this token brings is 64-bit arithmetic, the rest is what was there
    keys, values = s["keys"].double(), s["values"].double()
    mass, positions = s["mass"].clone(), s["positions"].clone()
    for head in range(2):
        new = head_of(rows[:, 8192 + 256 * head: 8448 + 256 * head], s["k_weight"])
        for lane, (n, position) in enumerate(s["lanes"].tolist()):
            at = (int(s["table"][lane, (n - 1) // s["page"]]), head, (n - 1) % s["page"])
            keys[at], values[at] = new[lane], rows[lane, 8704 + 256 * head: 8960 + 256 * head]
            mass[lane, head, n - 1], positions[lane, head, n - 1] = 0.0, position
    gate = torch.stack([rows[:, 512 * h + 256: 512 * h + 512] for h in range(16)], dim=1)
    return {"keys": keys, "values": values, "mass": mass, "positions": positions, "q": q, "gate": gate}


def exact(case, seed):
    if case["op"] not in ("decode", "rope"):
        return None      # rows are moved, nothing is computed
    state = prepare(case, seed)
    return _exact_decode(state) if case["op"] == "decode" else _exact_rope(state)
