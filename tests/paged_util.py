"""Plain 64-bit forms of the paged-cache operators, and batches to run them on."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step relative to the value
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step of the smallest values


class Batch:
    """Sequences of ``(new tokens, rows)`` in a pool whose unused rows are NaN; ``pages`` in random order."""

    def __init__(self, pkg, device, spans, *, heads, kv, dim, page, dtype, seed=0, spare=0, layout="heads", one_page=False):
        gen = torch.Generator().manual_seed(seed)
        self.spans, self.heads, self.kv, self.dim, self.page, self.dtype = spans, heads, kv, dim, page, dtype
        self.tokens = sum(t for t, _ in spans)
        self.total = self.tokens + spare
        rows = max([n for _, n in spans] + [1])
        self.width = 1 if one_page else -(-rows // page) + 1
        counts = [-(-n // page) for _, n in spans]
        pages = sum(counts) + 2
        order = torch.randperm(pages, generator=gen)
        table = torch.full((len(spans), self.width), -7, dtype=torch.int32)    # entries behind the last row are no pages
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = order[at:at + c].to(torch.int32)
            at += c
        self.host = {}
        for name in ("keys", "values"):
            pool = torch.full((pages, kv, page, dim), float("nan"), dtype=dtype)
            for b, (_, n) in enumerate(spans):
                for r in range(0, n, page):
                    m = min(page, n - r)
                    pool[table[b, r // page].item(), :, :m] = torch.randn((kv, m, dim), generator=gen).to(dtype)
            self.host[name] = pool
        self.query = torch.randn((self.total, heads, dim), generator=gen).to(dtype)
        self.table = table
        self.lengths = torch.tensor([n for _, n in spans], dtype=torch.int32)
        self.starts = torch.tensor([sum(t for t, _ in spans[:b]) for b in range(len(spans) + 1)], dtype=torch.int32)
        place = {"heads": lambda t: t.to(device),
                 "rows": lambda t: t.transpose(1, 2).contiguous().to(device).transpose(1, 2)}[layout]
        self.cache = pkg.ops.PagedKV(place(self.host["keys"]), place(self.host["values"]), table.to(device),
                                     self.lengths.to(device))
        self.q, self.s = self.query.to(device), self.starts.to(device)

    def rows(self, b, name="keys"):
        """Rows of sequence b, [rows, kv, dim], in 64 bits."""
        n = self.spans[b][1]
        pool = self.host[name].double()
        r = torch.arange(n)
        return pool[self.table[b, r // self.page].long(), :, r % self.page].reshape(n, self.kv, self.dim)


def attend(q, k, v, seen, scale):
    """One head: rows q [R, D] over k, v [n, D], row r over the first seen[r]; the result, the sum of weights times |v| and the
    largest sum of |q||k| over a row's keys.  Values that a row does not see take no part."""
    out, size, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for r in range(q.shape[0]):
        n = int(seen[r])
        if n == 0:
            continue
        p = torch.softmax(scale * (k[:n] @ q[r]), 0)
        out[r], size[r] = p @ v[:n], p @ v[:n].abs()
        most = max(most, float((k[:n].abs() @ q[r].abs()).max()))
    return out, size, most


def expected(batch, scale, causal, prefix=None):
    """(out, size, most, keys) over the covered tokens: see attend; keys: most keys of a row."""
    shape = (batch.tokens, batch.heads, batch.dim)
    out, size = torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)
    most, keys, at = 0.0, 1, 0
    group = batch.heads // batch.kv
    for b, (t, n) in enumerate(batch.spans):
        k, v, front = batch.rows(b), batch.rows(b, "values"), 0
        if prefix is not None:
            front = prefix.spans[0][1]
            k, v = torch.cat((prefix.rows(0), k)), torch.cat((prefix.rows(0, "values"), v))
        seen = front + (torch.arange(n - t, n) + 1 if causal else torch.full((t,), n)).clamp(min=0)
        for h in range(batch.heads):
            o, s, m = attend(batch.query[at:at + t, h].double(), k[:, h // group], v[:, h // group], seen, scale)
            out[at:at + t, h], size[at:at + t, h], most = o, s, max(most, m)
        keys, at = max(keys, front + n), at + t
    return out, size, most, keys


def bound(dtype, dim, scale, size, most, keys):
    """How far an output may be off, per element.

    A score's fp32 sum of ``dim`` exact products is off by at most ``dim 2^-24 sum |q||k|`` (times scale), scaling and exponent add
    three roundings of a number of at most ``scale sum |q||k| log2 e``: a weight is off by ``(dim + 6) 2^-24 scale most`` relative, plus
    2^-22 for the exponential, and so is the sum of weights it is divided by.  Sums over the keys and over the partial results add
    2^-24 a term.  The rounding of the weight and that of the output are off by half a step each.  All of it is relative to the sum
    of weights times |v|, but half a smallest step a weight.
    """
    weight = (dim + 6) * 2.0 ** -24 * scale * most + 2.0 ** -22
    relative = 2 * UNIT[dtype] * (1 + UNIT[dtype]) + 2 * weight + 2 * (keys + 16) * 2.0 ** -24
    return relative * size + (keys + 1) * TINY[dtype] * 8        # |v| stays under 8


def expected_wide(batch, scale, causal, device, prefix=None):
    """expected() on the device, a head at a time over all rows of a sequence (values must be finite)."""
    shape = (batch.tokens, batch.heads, batch.dim)
    out, size = torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)
    most, keys, at, group = 0.0, 1, 0, batch.heads // batch.kv
    for b, (t, n) in enumerate(batch.spans):
        k, v, front = batch.rows(b), batch.rows(b, "values"), 0
        if prefix is not None:
            front = prefix.spans[0][1]
            k, v = torch.cat((prefix.rows(0), k)), torch.cat((prefix.rows(0, "values"), v))
        seen = front + (torch.arange(n - t, n) + 1 if causal else torch.full((t,), n)).clamp(min=0)
        hidden = torch.arange(front + n)[None] >= seen[:, None]
        hidden, k, v = hidden.to(device), k.to(device), v.to(device)
        for h in range(batch.heads):
            q, kh, vh = batch.query[at:at + t, h].double().to(device), k[:, h // group].contiguous(), v[:, h // group].contiguous()
            p = torch.softmax((scale * (q @ kh.T.contiguous())).masked_fill(hidden, -float("inf")), 1).nan_to_num(0.0)
            out[at:at + t, h], size[at:at + t, h] = (p @ vh).cpu(), (p @ vh.abs()).cpu()
            if t and front + n:
                most = max(most, float((q.abs() @ kh.abs().T.contiguous()).masked_fill(hidden, 0.0).max()))
        keys, at = max(keys, front + n), at + t
    return out, size, most, keys


def turned(x, weight, inv_freq, positions, eps):
    """64-bit norm and rotation of rows x [tokens, heads, dim]."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + 1.0)
    if inv_freq is not None:
        a = positions.double()[:, None] * inv_freq.double()[None]
        c, s, h = a.cos()[:, None], a.sin()[:, None], inv_freq.shape[0]
        x = torch.cat((x[..., :h] * c - x[..., h:2 * h] * s, x[..., h:2 * h] * c + x[..., :h] * s, x[..., 2 * h:]), -1)
    return x
