"""Cases for the operators over K and V pages, and their definition in 64 bits."""
import math

import torch

PAGE = 64
TYPES = dict(bf16=torch.bfloat16, f16=torch.float16, e4m3=torch.float8_e4m3fn)


def nan_like(t):
    """All bits set: a NaN in each of the types."""
    t.view(torch.uint8).fill_(0xFF)


class Case:
    """Requests of kv_len[b] entries of which new[b] are the call's tokens; what no token of the call sees, and every page that no request holds, is NaN."""

    def __init__(self, kv_len, new, Hkv=2, G=4, D=64, dtype="bf16", q_dtype=None, window=0, first=0, sink=False, seed=0, packed=False, spare=2, fused=False, by=2.0, width=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dev = dict(device="cuda", generator=g)
        self.kv_len, self.B, self.Hkv, self.G, self.D, self.window, self.first = list(kv_len), len(kv_len), Hkv, G, D, window, first
        self.new = [new] * self.B if isinstance(new, int) else list(new)
        self.dtype, self.packed = TYPES[dtype], packed
        self.q_dtype = TYPES[q_dtype or ("bf16" if dtype == "e4m3" else dtype)]
        H = self.H = Hkv * G
        pages = max(max((n + PAGE - 1) // PAGE for n in kv_len), 1, width)
        P = self.B * pages + spare
        self.scales = [None, None]
        if dtype == "e4m3":
            self.scales = [0.03 + 0.03 * torch.rand(Hkv, **dev) for _ in "kv"]
        self.pools = [(torch.randn(P, PAGE, Hkv, D, **dev) * (20 if dtype == "e4m3" else 1)).to(self.dtype) for _ in "kv"]
        order = torch.randperm(P, **dev).int()
        self.table = torch.full((self.B, pages), -1, device="cuda", dtype=torch.int32)
        self.start = [0]
        for n in self.new:
            self.start.append(self.start[-1] + n)
        for b, n in enumerate(self.kv_len):
            held = (n + PAGE - 1) // PAGE
            self.table[b, :held] = order[b * pages:b * pages + held]
        seen = torch.zeros(P, PAGE, dtype=torch.bool, device="cuda")
        for b in range(self.B):
            v = self.visible(b).any(0)
            if v.numel():
                at = torch.arange(v.numel(), device="cuda")[v]
                seen[self.table[b, at // PAGE].long(), at % PAGE] = True
        for pool in self.pools:
            x = pool.view(torch.uint8).reshape(P, PAGE, -1)
            x[~seen] = 0xFF
        rows = self.start[-1]
        wide = H + 2 * Hkv if fused else H
        q = (torch.randn(rows, wide, D, **dev) * by).to(self.q_dtype)[:, :H]
        self.q = q if packed else q.unflatten(0, (self.B, self.new[0]))
        self.sink = torch.randn(H, **dev) * 2 if sink else None
        self.scale = D ** -0.5
        self.len_t = torch.tensor(self.kv_len, device="cuda", dtype=torch.int32)
        self.start_t = torch.tensor(self.start, device="cuda", dtype=torch.int32)

    def visible(self, b):
        """bool [new[b], kv_len[b]]"""
        n, T = self.kv_len[b], self.new[b]
        p = torch.arange(n - T, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        v = j <= p
        return v & ((p - j < self.window) | (j < self.first)) if self.window else v

    def args(self):
        return (*self.pools, self.table, self.len_t, self.scale), dict(window=self.window, first=self.first, k_scale=self.scales[0], v_scale=self.scales[1], attn_sink=self.sink)

    def call(self, d, **more):
        a, kw = self.args()
        if self.packed:
            return d.gqa_prefill(self.q, self.start_t, *a, **kw, **more)
        return d.gqa_decode(self.q, *a, **kw, **more)

    def entries(self, i, b):
        n = self.kv_len[b]
        pool = self.pools[i]
        rows = pool.view(torch.uint8)[self.table[b, :(n + PAGE - 1) // PAGE].long()].view(pool.dtype).flatten(0, 1)[:n].double()
        rows = torch.where(self.visible(b).any(0)[:, None, None], rows, 0.0)
        return rows if self.scales[i] is None else rows * self.scales[i].double()[:, None]

    def expected(self):
        """out, lse, weights [B][kv_len], in 64 bits, and bounds of what the kernels' roundings may make of them."""
        q = self.q.reshape(-1, self.H, self.D).double()
        rows = q.shape[0]
        out = torch.zeros(rows, self.H, self.D, device="cuda", dtype=torch.float64)
        lse = torch.full((rows, self.H), -math.inf, device="cuda", dtype=torch.float64)
        out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
        weights, weight_tol = [], []
        half = torch.finfo(self.q_dtype).eps / 2                       # of a rounding of the output
        # P is rounded to the type that V is multiplied in: half a step, eps / 2 of each weight.  An 8-bit cache is read as FP16 by the decode kernel; for prompts it is
        # brought to the type of the queries, so that with BF16 ones P is rounded to BF16 there: 2^-8 of a weight instead of 2^-11
        p_half = torch.finfo(self.dtype if self.dtype != torch.float8_e4m3fn else self.q_dtype if self.packed else torch.float16).eps / 2
        # P in FP16: below its normal numbers a weight is off by up to 2^-25 of the largest one
        p_small = 0.0 if self.dtype == torch.bfloat16 else 2.0 ** -25
        # BF16 queries over an 8-bit cache: elements below 2^-14 of the row's largest are off by up to 2^-25 of it
        q_small = 2.0 ** -25 if self.dtype == torch.float8_e4m3fn and self.q_dtype == torch.bfloat16 else 0.0
        for b in range(self.B):
            lo, hi = self.start[b], self.start[b + 1]
            k, v, see = self.entries(0, b), self.entries(1, b), self.visible(b)
            w, wt = torch.zeros(self.kv_len[b], device="cuda", dtype=torch.float64), torch.zeros(self.kv_len[b], device="cuda", dtype=torch.float64)
            for h in range(self.H if hi > lo and self.kv_len[b] > 0 else 0):
                kh, vh, qh = k[:, h // self.G], v[:, h // self.G], q[lo:hi, h]
                x = (qh @ kh.T * self.scale).masked_fill(~see, -math.inf)
                total = torch.logsumexp(x, -1)
                whole = total if self.sink is None else torch.logaddexp(total, self.sink[h].double())
                p = torch.exp(x - whole[:, None]).nan_to_num(0.0)
                out[lo:hi, h], lse[lo:hi, h] = p @ vh, total
                # a score is a sum of D products in 32 bits (each addition rounds by 2^-24 of the partial sum), scaled (2 roundings), exponentiated (2^-22 and a difference
                # of numbers of its size); sums of the weights add 32 such roundings at most in a row of a warp's parts
                size = (qh.abs() @ kh.abs().T * self.scale).masked_fill(~see, 0.0)
                off = (self.D * 2.0 ** -24 + 3 * 2.0 ** -24) * size + q_small * self.scale * qh.abs().amax(-1, keepdim=True) * kh.abs().sum(-1) + 2.0 ** -20
                worst = off.amax(-1) + 2.0 ** -19
                pv = p @ vh.abs()
                top = torch.exp(x.amax(-1) - whole).nan_to_num(0.0)
                out_tol[lo:hi, h] = (p_half + 2 * worst[:, None]) * pv + p_small * top[:, None] * (see.double() @ vh.abs()) + half * out[lo:hi, h].abs() * 1.01 + 1e-7
                lse_tol[lo:hi, h] = worst + 2.0 ** -22 * total.abs().nan_to_num(0.0, 0.0, 0.0)
                w += p.sum(0)
                wt += (p * (off + worst[:, None])).sum(0)
            weights.append(w)
            weight_tol.append(wt + 2.0 ** -23 * w * 8)
        if self.q_dtype == torch.float16:
            out_tol += 2.0 ** -24                                      # FP16's steps near 0
        return out, lse, weights, out_tol, lse_tol, weight_tol

    def check(self, out, lse, weights=None, before=None):
        want, want_lse, want_w, tol, lse_tol, w_tol = self.expected()
        got, got_lse = out.reshape(want.shape).double(), lse.reshape(want_lse.shape).double()
        assert torch.equal(torch.isneginf(got_lse), torch.isneginf(want_lse)), "rows that see nothing"
        none = torch.isneginf(want_lse)
        assert (got[none] == 0).all(), "a row that sees nothing gives 0"
        err = (got - want).abs()
        bad = ~(err <= tol)
        assert not bad.any(), f"out: {int(bad.sum())} of {bad.numel()} off, by up to {float(err[bad].nan_to_num(9e9).max()):.3e}, first at {bad.nonzero()[0].tolist()}, of tolerance {float((err / tol).nan_to_num(9e9).max()):.2f}"
        diff = torch.where(none, 0.0, got_lse - want_lse).abs()
        assert (diff <= lse_tol).all(), f"lse off by {float(diff.max()):.3e}, {float((diff / lse_tol).nan_to_num(0).max()):.2f} of the tolerance"
        if weights is not None:
            for b, n in enumerate(self.kv_len):
                got_w = (weights[b, :n] - before[b, :n]).double()
                diff = (got_w - want_w[b]).abs()
                allowed = w_tol[b] + 2.0 ** -23 * (before[b, :n].double().abs() + want_w[b])        # (the sum of old and new rounds, and so does the difference here)
                assert (diff <= allowed).all(), f"weights of request {b} off by {float(diff.max()):.3e}, {float((diff / allowed).max()):.2f} of the tolerance"
                assert torch.equal(weights[b, n:], before[b, n:])
