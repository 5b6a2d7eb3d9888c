"""A paged cache for the tests, its 64-bit definitions and the bounds that the tests hold the kernels to."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative


class Cache:
    """Pools with the lanes' pages scattered, spare pages, and not-a-number in every row that holds no token."""

    def __init__(self, lens, kv_heads, dim, dtype=torch.bfloat16, page=16, slot_major=False, spare=3, extra_columns=2, seed=0,
                 device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.gen, self.page, self.device = gen, page, device
        per_lane = [-(-n // page) for n in lens]
        columns = max(per_lane) + extra_columns
        pages = len(lens) * columns + spare
        order = torch.randperm(pages, generator=gen, device=device, dtype=torch.int32)
        self.table = order[: len(lens) * columns].reshape(len(lens), columns).contiguous()
        self.spare = order[len(lens) * columns:].long()
        shape = (pages, page, kv_heads, dim) if slot_major else (pages, kv_heads, page, dim)
        pools = [torch.randn(shape, generator=gen, device=device).to(dtype) for _ in range(2)]
        self.keys, self.values = (p.permute(0, 2, 1, 3) if slot_major else p for p in pools)
        for pool in (self.keys, self.values):
            pool[self.spare] = float("nan")
            for lane, n in enumerate(lens):
                for column in range(columns):
                    first = max(0, n - column * page)
                    if first < page:
                        pool[int(self.table[lane, column]), :, first:] = float("nan")
        self.lens = list(lens)
        self.lanes = torch.tensor([[n, max(0, n - 1)] for n in lens], dtype=torch.int32, device=device)
        self.mass = torch.rand((len(lens), kv_heads, columns * page), generator=gen, device=device)
        slots = torch.arange(columns * page, dtype=torch.int32, device=device)
        self.positions = slots.expand(len(lens), kv_heads, -1).contiguous()

    def rows(self, pool, lane, head, n):
        s = torch.arange(n, device=self.device)
        return pool[self.table[lane, s // self.page].long(), head, s % self.page]

    def clone(self):
        other = object.__new__(Cache)
        other.__dict__.update(self.__dict__)
        for name in ("table", "lanes", "mass", "positions"):
            setattr(other, name, getattr(self, name).clone())
        for name in ("keys", "values"):
            src = getattr(self, name)
            setattr(other, name, torch.empty_strided(src.shape, src.stride(), dtype=src.dtype, device=src.device).copy_(src))
        return other


def decode_definition(cache, q, gate, scale):
    """out, its bound, the weights added to the mass and their bound, in 64 bits.

    Bound of an output: the result is rounded once (half a step of it); the weights are rounded to the cache's type before
    the product with V (half a step of each: of sum p |v|); scores are f32 sums of dim products, each term off by at most
    (dim + 2) 2^-24 of sum |q k| scale, which the exponential turns into that relative error of a weight (twice: numerator and
    sum); sums over n slots run over at most n / 64 + 80 additions; exp2 and the final division add a few last places."""
    u, dim = U[q.dtype], q.shape[2]
    heads = cache.keys.shape[1]
    group = q.shape[1] // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    added = torch.zeros(cache.mass.shape, dtype=torch.float64, device=q.device)
    added_bound = torch.zeros_like(added)
    for lane, n in enumerate(cache.lanes[:, 0].tolist()):
        for head in range(heads if n else 0):
            k, v = (cache.rows(x, lane, head, n).double() for x in (cache.keys, cache.values))
            of = slice(head * group, (head + 1) * group)
            x = q[lane, of].double()
            p = torch.softmax(x @ k.T * scale, dim=-1)
            size = float((x.abs() @ k.abs().T).max()) * abs(scale)
            slack = 2 * (dim + 2) * 2.0 ** -24 * size + (n / 64 + 80) * 2.0 ** -24 + 2.0 ** -20
            o, a = p @ v, p @ v.abs()
            if gate is not None:
                s = torch.sigmoid(gate[lane, of].double())
                o, a = o * s, a * s
            out[lane, of] = o
            # 2^-25: below it f16 has no normal step left (weights under 2^-14 of the largest one round to multiples of 2^-24)
            tiny = 2.0 ** -25 * v.abs().sum(dim=0) if q.dtype == torch.float16 else 0.0
            bound[lane, of] = u * o.abs() + (u + slack) * a + tiny + 2.0 ** -24
            added[lane, head, :n] = p.sum(dim=0)
            added_bound[lane, head, :n] = slack * p.sum(dim=0) + 2.0 ** -126
    return out, bound, added, added_bound


def evict_definition(cache, keep, sink, recent):
    """The cache after an eviction: lane by lane and head by head, nothing vectorised."""
    after = cache.clone()
    for lane, (n, position) in enumerate(cache.lanes.tolist()):
        if n <= keep:
            continue
        for head in range(cache.keys.shape[1]):
            mass = cache.mass[lane, head, :n].tolist()
            where = cache.positions[lane, head, :n].tolist()

            def rank(s):
                if s < sink or where[s] + recent > position:
                    return (0, 0.0, s)
                return (2, 0.0, s) if mass[s] != mass[s] else (1, -mass[s], s)
            kept = set(sorted(range(n), key=rank)[:keep])
            holes = [s for s in range(keep) if s not in kept]
            donors = [s for s in range(keep, n) if s in kept]
            assert len(holes) == len(donors)
            if not holes:
                continue
            to, origin = (torch.tensor(x, device=cache.device) for x in (holes, donors))
            for pool_after, pool in ((after.keys, cache.keys), (after.values, cache.values)):
                pool_after[cache.table[lane, to // cache.page].long(), head, to % cache.page] = \
                    pool[cache.table[lane, origin // cache.page].long(), head, origin % cache.page]
            for plane_after, plane in ((after.mass, cache.mass), (after.positions, cache.positions)):
                plane_after[lane, head, to] = plane[lane, head, origin]
    return after


def same(a, b):
    """Bit for bit, not-a-number included."""
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return bool(torch.equal(a.contiguous().view(kind), b.contiguous().view(kind)))


def same_cache(a, b):
    return all(same(getattr(a, x), getattr(b, x)) for x in ("keys", "values", "mass", "positions", "lanes", "table"))
