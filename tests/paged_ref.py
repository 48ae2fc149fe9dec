"""Plain forms of the batched-serving operators for the tests: 64-bit
attention over a paged cache, the cache's formats, the sampler in whole
numbers."""
import torch

F16, Q8_0 = 1, 2


def quantise(x):
    """Q8_0 of fp32 x's last dimension: (codes int8, scales half)."""
    b = x.float().unflatten(-1, (-1, 32))
    mx = torch.nan_to_num(b.abs(), nan=0.0, posinf=float("inf")).amax(-1)
    d = (mx / torch.full_like(mx, 127.0)).clamp(max=65504.0).half()
    df = d.float().unsqueeze(-1)
    code = torch.where(df > 0, (b / df).round().clamp(-127, 127), torch.zeros_like(b))
    return torch.nan_to_num(code, nan=0.0).to(torch.int8).flatten(-2), d


def rope(x, cs):
    """x [tokens][heads][hd] rotated by cs [tokens][hd] ({cos, sin} pairs)."""
    a, b = x.unflatten(-1, (-1, 2)).unbind(-1)
    c, s = cs.unflatten(-1, (-1, 2)).unbind(-1)
    c, s = c[:, None], s[:, None]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


class Cache:
    """Pools whose free pages, and the rows past each sequence's end, hold NaN
    (F16, and the scales of Q8_0)."""

    def __init__(self, gb, dtype, n_kv, hd, page, kv_lens, seed, fill=True, spare=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.n_kv, self.hd, self.page, self.kv_lens = dtype, n_kv, hd, page, list(kv_lens)
        need = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((max(1, len(need)), max(need + [0]) + 2), -7, dtype=torch.int32, device="cuda")
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at: at + n]
            at += n
        nbytes = gb.kv_page_bytes(dtype, n_kv, hd, page)
        self.pools = [torch.full((self.n_pages * nbytes // 2,), 0x7E00, dtype=torch.int16, device="cuda")
                      .view(torch.uint8).view(self.n_pages, n_kv, -1) for _ in range(2)]
        self.len = torch.tensor(self.kv_lens, dtype=torch.int32, device="cuda")
        self.h = gb.KVCache(dtype, n_kv, hd, page, self.n_pages, *self.pools)
        # values of every sequence, fp64 [kv_len][n_kv][hd]
        self.k, self.v = [], []
        if fill:
            for s, n in enumerate(self.kv_lens):
                for pool, kept in zip(self.pools, (self.k, self.v)):
                    x = torch.randn(n, n_kv, hd, generator=g, device="cuda")
                    kept.append(self.put(pool, s, x))

    def parts(self, pool):
        p, hd = self.page, self.hd
        if self.dtype == F16:
            return pool.view(torch.float16).unflatten(-1, (p, hd)), None
        return (pool[..., : p * hd].view(torch.int8).unflatten(-1, (p, hd)),
                pool[..., p * hd:].view(torch.float16).unflatten(-1, (p, hd // 32)))

    def put(self, pool, s, x):
        rows, scales = self.parts(pool)
        pos = torch.arange(x.shape[0], device="cuda")
        pg, r = self.table[s, pos // self.page].long(), pos % self.page
        if scales is None:
            rows[pg, :, r] = x.half()
            return x.half().double()
        codes, d = quantise(x)
        rows[pg, :, r] = codes
        scales[pg, :, r] = d
        return (codes.double().unflatten(-1, (-1, 32)) * d.double().unsqueeze(-1)).flatten(-2)

    def get(self, pool, s, n):
        rows, scales = self.parts(pool)
        pos = torch.arange(n, device="cuda")
        pg, r = self.table[s, pos // self.page].long(), pos % self.page
        x = rows[pg, :, r].double()
        if scales is None:
            return x
        return (x.unflatten(-1, (-1, 32)) * scales[pg, :, r].double().unsqueeze(-1)).flatten(-2)


def attention(q, cache, q_lens):
    """fp64 [tokens][heads * hd]: token i of sequence s sees positions up to
    kv_len - q_len + i; none: zeros."""
    out, t0, hd, kv = [], 0, cache.hd, cache.n_kv
    for s, n in enumerate(q_lens):
        m = cache.kv_lens[s]
        x = q[t0: t0 + n].double().reshape(n, kv, q.shape[1] // (kv * hd), hd)
        t0 += n
        if m == 0 or n == 0:
            out.append(torch.zeros(n, q.shape[1], dtype=torch.float64, device=q.device))
            continue
        sc = torch.einsum("nghd,mgd->nghm", x, cache.k[s]) / hd ** 0.5
        hid = torch.arange(m, device=q.device)[None] > torch.arange(m - n, m, device=q.device)[:, None]
        sc = sc.masked_fill(hid[:, None, None], float("-inf"))
        p = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0)
        out.append(torch.einsum("nghm,mgd->nghd", p, cache.v[s]).reshape(n, -1))
    return torch.cat(out) if out else q.double()


def share(total, part):
    return (total >> 24) * part + (((total & 0xFFFFFF) * part) >> 24)


def sample_row(row, temperature, top_k, top_p, min_p, u):
    """The definition in Python integers (row: fp32 CUDA tensor; the fp32
    exponential is the device's)."""
    x = torch.nan_to_num(row, nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    mx = x.max()
    if mx == float("-inf"):
        return -1
    order = torch.sort(x, descending=True, stable=True).indices.tolist()
    if not temperature > 0:
        return order[0]
    t = torch.full_like(x, temperature)
    e = torch.where(x == mx, torch.ones_like(x), torch.exp((x - mx) / t))
    w = (e.double() * 2.0 ** 40).round().to(torch.int64).tolist()
    e = e.tolist()
    if top_k > 0:
        order = order[:top_k]
    total = sum(w[i] for i in order)
    kept, run = [], 0
    if top_p < 1:
        f32 = torch.tensor(max(top_p, 0.0), dtype=torch.float32).item()
        goal = share(total, round(f32 * 2 ** 24))
        for j, i in enumerate(order):
            if j and run >= goal:
                break
            kept.append(i)
            run += w[i]
    else:
        kept = order
    if min_p > 0:
        least = torch.tensor(min(min_p, 1.0), dtype=torch.float32).item()
        kept = [i for i in kept if e[i] >= least]
    target = share(sum(w[i] for i in kept), min(int(u * 2 ** 24), 2 ** 24 - 1))
    run = 0
    for i in sorted(kept):
        run += w[i]
        if run > target:
            return i
    raise AssertionError("nothing drawn")
