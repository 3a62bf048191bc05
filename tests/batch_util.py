"""Plain 64-bit forms of the operators of a batch's states and drafts, and batches to run them on."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step relative to the value
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step of the smallest values
EPS = 2.0 ** -24


class Layer:
    """A GDN layer's block of ``spans`` tokens a sequence, with ``spare`` tokens behind the last; states in a pool of shuffled
    slots among others'.  ``missing``: sequences without a slot, ``fresh``: that start from zeros, ``counts``: None or tokens to
    advance by."""

    def __init__(self, pkg, device, spans, *, key_heads=2, value_heads=4, dim=128, dtype=torch.bfloat16, seed=0, spare=0,
                 missing=(), fresh=(), counts=None, raw_gates=True, gates_dtype=None, strided=True, decay_scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        normal = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
        self.pkg, self.device, self.spans, self.dtype = pkg, device, list(spans), dtype
        self.hk, self.hv, self.dim = key_heads, value_heads, dim
        self.channels = dim * (2 * key_heads + value_heads)
        b, total = len(spans), sum(spans) + spare
        self.total, self.tokens = total, sum(spans)
        pool = b + 3
        self.slots = torch.randperm(pool, generator=gen)[:b].to(torch.int32)
        missing, fresh = ([i for i in v if i < b] for v in (missing, fresh))
        for i in missing:
            self.slots[i] = (-1, pool, -2 ** 31, 2 ** 31 - 1)[i % 4]
        self.starts = torch.tensor([sum(spans[:i]) for i in range(b + 1)], dtype=torch.int32)
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
        self.fresh = torch.tensor([i in fresh for i in range(b)]) if len(fresh) else None
        self.history = normal(pool, self.channels, 3).to(dtype)
        self.recurrent = normal(pool, value_heads, dim, dim) * 0.3
        for i in fresh:   # a slot that a fresh sequence does not read may hold anything
            if 0 <= int(self.slots[i]) < pool:
                self.history[int(self.slots[i])], self.recurrent[int(self.slots[i])] = math.nan, math.nan
        self.weight = (normal(self.channels, 1, 4) * 0.4).to(dtype)
        width = self.channels + value_heads * dim + 2 * value_heads
        pad = -width % 8
        proj = normal(total, width + pad).to(dtype)
        mixed = torch.nn.functional.silu(normal(total, self.channels)).to(dtype)
        gates = normal(2, total, value_heads)
        self.a_log, self.dt_bias = (torch.rand((value_heads,), generator=gen) * 3.0 - 2.0), normal(value_heads)
        if raw_gates:
            decay, beta = gates
        else:
            self.a_log = self.dt_bias = None
            decay, beta = -gates[0].abs() * decay_scale, torch.sigmoid(gates[1])
        kind = gates_dtype or (dtype if raw_gates else torch.float32)
        self.decay, self.beta = decay.to(kind), beta.to(kind)
        # on the device: views of one projection's rows, as a layer has them, or tensors of their own
        dev = lambda t: None if t is None else t.to(device)  # noqa: E731
        kw, vw = key_heads * dim, value_heads * dim
        self.x = proj[:, :self.channels]
        self.query, self.key, self.value = (t.unflatten(-1, (-1, dim)) for t in mixed.split((kw, kw, vw), -1))
        self.d = {n: dev(getattr(self, n)) for n in ("slots", "starts", "counts", "fresh", "history", "recurrent", "weight", "a_log", "dt_bias",
                                                     "decay", "beta")}
        if strided:
            rows = dev(proj)
            self.d["x"] = rows[:, :self.channels]
            whole = dev(mixed)
            self.d["query"], self.d["key"], self.d["value"] = (t.unflatten(-1, (-1, dim)) for t in whole.split((kw, kw, vw), -1))
            wide = torch.cat((self.d["decay"], self.d["beta"]), 1)
            self.d["decay"], self.d["beta"] = wide[:, :value_heads], wide[:, value_heads:]
        else:
            self.d |= {n: dev(getattr(self, n).contiguous()) for n in ("x", "query", "key", "value")}
        self.pool = pkg.ops.StatePool(self.d["history"], self.d["recurrent"], self.d["slots"])

    def has_slot(self, b):
        return 0 <= int(self.slots[b]) < self.history.shape[0]

    def advanced(self, b):
        n = self.spans[b]
        c = n if self.counts is None else min(max(int(self.counts[b]), 0), n)
        return c if self.has_slot(b) else 0

    def starts_from_zeros(self, b):
        return not self.has_slot(b) or (self.fresh is not None and bool(self.fresh[b]))

    def memory(self, b):
        """Tokens that the slowest head of sequence b remembers: sum of e^(g summed behind them)."""
        at, n = int(self.starts[b]), self.advanced(b)
        g = self.decay[at:at + n].double()
        if self.a_log is not None:
            g = -self.a_log.double().exp() * torch.nn.functional.softplus(g + self.dt_bias.double())
        later = g.flip(0).cumsum(0)
        return 1.0 + float(later.exp().sum(0).max())

    # -- calls
    def conv(self, out=None, **kw):
        d = self.d
        return self.pkg.ops.gdn_conv(d["x"], d["weight"], self.pool, d["starts"], fresh=d["fresh"], counts=d["counts"], out=out, **kw)

    def rule(self, out=None, **kw):
        d = self.d
        return self.pkg.ops.gdn_rule(d["query"], d["key"], d["value"], d["decay"], d["beta"], self.pool, d["starts"], a_log=d["a_log"],
                                     dt_bias=d["dt_bias"], fresh=d["fresh"], counts=d["counts"], out=out, **kw)

    def advance(self, **kw):
        d = self.d
        self.pkg.ops.gdn_advance(self.pool, d["x"], d["key"], d["value"], d["decay"], d["beta"], d["starts"], d["counts"], a_log=d["a_log"],
                                 dt_bias=d["dt_bias"], fresh=d["fresh"], **kw)

    # -- 64 bits
    def expected_conv(self):
        """(out, sum of |weight x|) over the covered tokens, and the histories afterwards (their own bits)."""
        w = self.weight.double()[:, 0]
        out, size, history = [], [], self.history.clone()
        for b, n in enumerate(self.spans):
            at = int(self.starts[b])
            before = torch.zeros((3, self.channels), dtype=self.dtype) if self.starts_from_zeros(b) else self.history[int(self.slots[b])].t()
            line = torch.cat((before, self.x[at:at + n]))
            wide = line.double()
            y = sum(wide[j:j + n] * w[:, j] for j in range(4))
            size.append(sum((wide[j:j + n] * w[:, j]).abs() for j in range(4)))
            out.append(y * torch.sigmoid(y))
            c = self.advanced(b)
            if c:
                history[int(self.slots[b])] = line[c:c + 3].t()
        none = torch.zeros((0, self.channels), dtype=torch.float64)
        return torch.cat([none, *out]), torch.cat([none, *size]), history

    def expected_rule(self, normalise=True, scale=None):
        """Outputs, states, and bounds of what fp32 arithmetic may be off in both.

        A column of the state is off by a vector e with e' = e^g (I - beta k k^T) e + (what the token itself adds), and a unit key
        and beta <= 1 make that product a contraction: |e'| <= e^g |e| + local.  local: a product of a column and the key is
        off by dim EPS of its size (as a sum of dim terms, or of the chunk's at most 64 earlier keys' products); solving for the
        chunk's u and adding them up adds at most 4 * 64 + 64 roundings of u, v and the column; the gates are off by a few steps of
        theirs, a decay e^g by |g| times that.  An output is off by e times |q| and as many roundings of its own product.
        """
        d, rep = self.dim, self.hv // self.hk
        scale = d ** -0.5 if scale is None else scale
        recurrent, bound_s = self.recurrent.double().clone(), torch.zeros((*self.recurrent.shape[:2], d), dtype=torch.float64)
        outs, bounds = [], []
        local = (d + 5 * 64) * EPS
        for b, n in enumerate(self.spans):
            at = int(self.starts[b])
            s = (torch.zeros((self.hv, d, d), dtype=torch.float64) if self.starts_from_zeros(b)
                 else self.recurrent[int(self.slots[b])].double())
            e = torch.zeros((self.hv, d), dtype=torch.float64)
            out, bound = torch.zeros((n, self.hv, d), dtype=torch.float64), torch.zeros((n, self.hv, d), dtype=torch.float64)
            q, k = (t[at:at + n].double().repeat_interleave(rep, 1) for t in (self.query, self.key))
            if normalise:
                q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
            q, v = q * scale, self.value[at:at + n].double()
            g, beta = self.decay[at:at + n].double(), self.beta[at:at + n].double()
            if self.a_log is not None:
                g = -self.a_log.double().exp() * torch.nn.functional.softplus(g + self.dt_bias.double())
                beta = torch.sigmoid(beta)
            for t in range(n):
                fade = g[t].exp()[:, None]
                s = fade[..., None] * s
                size = s.norm(dim=1)
                u = beta[t][:, None] * (v[t] - (s * k[t][..., None]).sum(1))
                s = s + k[t][..., None] * u[:, None, :]
                gate = 8 * EPS * (1 + torch.where(g[t].isfinite(), g[t].abs(), 0.0))[:, None]   # e^-inf is exactly 0
                e = fade * e + (local + gate) * (size + beta[t][:, None] * v[t].abs() + u.abs())
                out[t] = (s * q[t][..., None]).sum(1)
                bound[t] = q[t].norm(dim=-1)[:, None] * (e + (local + gate) * (s.norm(dim=1) + size + u.abs()))
                if t + 1 == self.advanced(b):
                    recurrent[int(self.slots[b])], bound_s[int(self.slots[b])] = s, e
            outs.append(out)
            bounds.append(bound + UNIT[self.dtype] * (out.abs() + bound) + TINY[self.dtype])
        none = torch.zeros((0, self.hv, d), dtype=torch.float64)
        return torch.cat([none, *outs]), torch.cat([none, *bounds]), recurrent, bound_s

    def check_conv(self, got, what=""):
        """fp32: four products and three sums, exponential (a few steps and |y| steps of it), division; SiLU's slope is at most 1.1."""
        want, size, history = self.expected_conv()
        limit = 1.1 * 8 * EPS * size + want.abs() * (UNIT[self.dtype] * 1.01 + 16 * EPS * (1 + size)) + TINY[self.dtype]
        over = ((got[:self.tokens].double().cpu() - want).abs() - limit)
        assert not over.numel() or float(over.max()) <= 0, (what, float(over.max()))
        assert same_bits(self.d["history"].cpu(), history), what

    def check_state(self, want, bound, what=""):
        got = self.d["recurrent"].cpu()
        for b in range(len(self.spans)):
            if not self.has_slot(b):
                continue
            slot = int(self.slots[b])
            if self.advanced(b) == 0:
                assert same_bits(got[slot], self.recurrent[slot]), (what, "state that does not advance", b)
                continue
            off = (got[slot].double() - want[slot]).norm(dim=1)
            assert bool((off <= bound[slot] + EPS * want[slot].norm(dim=1)).all()), (what, b, float((off - bound[slot]).max()))
            # Over all columns roundings act independently.  A token rounds the state at most three times (decay, product, sum), each off
            # by at most EPS, and what it rounds away is remembered as the state is: over N tokens of memory 3 sqrt(N) EPS.  16 EPS beside
            # that: of the gates (|g| N < 1 steps of theirs), norms and the products of one token or chunk.
            limit = (16 + 3 * min(self.advanced(b), self.memory(b)) ** 0.5) * EPS
            assert float((got[slot].double() - want[slot]).norm()) <= limit * float(want[slot].norm()), (what, b)
        held = {int(s) for s in self.slots}
        for slot in range(got.shape[0]):
            if slot not in held:
                assert same_bits(got[slot], self.recurrent[slot]), (what, "another's slot", slot)

    def check_rule(self, got, what="", **kw):
        want, limit, recurrent, bound = self.expected_rule(**kw)
        over = (got[:self.tokens].double().cpu() - want).abs() - limit
        assert not over.numel() or float(over.max()) <= 0, (what, float(over.max()))
        self.check_state(recurrent, bound, what)


def same_bits(a, b):
    view = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.shape == b.shape and bool((a.contiguous().view(view) == b.contiguous().view(view)).all())


# ------------------------------------------------------------------ drafts
def chances(logits, temperature):
    """Probabilities of one row in 64 bits, zeros where it has nothing to give."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    top = x.max()
    if top == -math.inf:
        return torch.zeros_like(x)
    if not temperature > 0:
        return (torch.arange(x.numel()) == int((x == top).nonzero()[0])).double()
    w = torch.where(x == top, 1.0, torch.where(x == -math.inf, 0.0, ((x - top) / min(max(temperature, 1e-30), 1e30)).exp()))
    return w / w.sum()


def drawn(weights, uniform):
    total = weights.cumsum(0)
    over = ((total > uniform * total[-1]) & (weights > 0)).nonzero()
    held = (weights > 0).nonzero()
    return int(over[0]) if len(over) else int(held[-1]) if len(held) else -1


def verified(target, drafted, starts, uniforms, draft=None, temperature=None):
    """accepted and token of every sequence, and how near the nearest comparison was (of acceptance tests and of draws)."""
    accepted, token, margin = [], [], 1.0
    for b in range(len(starts) - 1):
        row, end = int(starts[b]), int(starts[b + 1])
        if row >= end:
            accepted.append(0), token.append(-1)
            continue
        t = 1.0 if temperature is None else float(temperature[b])
        first = row
        while True:
            p, x, u = chances(target[row], t), int(drafted[row]), float(uniforms[row])
            if row + 1 == end:
                left = p
                break
            inside = 0 <= x < p.numel()
            if draft is None or not t > 0:
                q = torch.zeros_like(p)
                if inside:
                    q[x] = 1.0
                qx = 1.0
            else:
                q = chances(draft[row], t)
                qx = float(q[x]) if inside else 0.0
            px = float(p[x]) if inside else 0.0
            if not u * qx < px:
                left = (p - q).clamp(min=0.0)
                u = float(uniforms[row + 1])
                break
            margin = min(margin, abs(px - u * qx) / max(px, 1e-300))
            row += 1
        if float(left.sum()) == 0.0:
            left = p
        total = left.cumsum(0)
        if float(total[-1]) > 0 and 0 <= u < 1:
            margin = min(margin, float(((total - u * total[-1]).abs() / total[-1])[left > 0].min()))
        accepted.append(row - first)
        token.append(drawn(left, u))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(token, dtype=torch.int32), margin
