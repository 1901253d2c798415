"""Inputs and bounds of the tests of attention over a step's rows and of rotations."""

import torch

from oracle import attend as OA

DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Step:
    """A step's requests [(tokens after it, rows)], behind shared prefixes (their lengths and which one each request is behind), over
    random pages of 8 bits, all on the CPU. Scales 2^-8 .. 2^-4, of either sign with signed. pad: rows past the last request's;
    lead: rows before the first."""

    def __init__(self, reqs, Hq, Hkv, D, fmt, seed, shared=(), of=None, prefix=None, pad=0, lead=0, signed=False, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.Hq, self.Hkv, self.D, self.fmt = Hq, Hkv, D, fmt
        self.lens = [n for n, _ in reqs]
        self.starts = [lead]
        for _, a in reqs:
            self.starts.append(self.starts[-1] + a)
        self.rows = self.starts[-1] + pad
        self.shared_lens, self.of, self.prefix = list(shared) or None, of, prefix
        need = [(max(n, 0) + 63) // 64 for n in self.lens] + [(n + 63) // 64 for n in shared]
        order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
        width = width or max(1, *need)
        table = torch.full((len(need), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table[:len(reqs)].contiguous()
        self.shared_table = table[len(reqs):].contiguous() if shared else None
        P = order.numel()
        self.k, self.v = (self.codes(g, P) for _ in "kv")
        self.ks, self.vs = (torch.exp2(torch.rand(P, Hkv, generator=g) * 4 - 8) for _ in "kv")
        if signed:
            self.ks, self.vs = (x * (torch.randint(0, 2, x.shape, generator=g) * 2 - 1) for x in (self.ks, self.vs))
        self.q = torch.randn(self.rows, Hq, D, generator=g).to(torch.bfloat16)
        self.scale = D ** -0.5

    def codes(self, g, P):
        x = torch.randn(P, self.Hkv, 64, self.D, generator=g)
        if self.fmt == "int8":
            return (x * 40).round().clamp(-127, 127).to(torch.int8)
        return (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)

    def i32(self, x):
        return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")

    def plan(self, window=0, max_rows=0):
        from kvskip_amd import kvskip as K

        cu = lambda t: None if t is None else t.cuda()
        sh = self.shared_lens is not None
        return K.attend_plan(self.i32(self.starts), self.i32(self.lens), self.rows, cu(self.table), self.Hq, self.Hkv,
                             max_rows=max_rows, window=window, prefix_lens=self.i32(self.prefix),
                             shared_table=cu(self.shared_table), shared_lens=self.i32(self.shared_lens) if sh else None,
                             shared_of=self.i32(self.of) if sh else None)

    def call(self, plan, softcap=0.0, slopes=None):
        from kvskip_amd import kvskip as K

        return K.attend(self.q.cuda(), self.k.cuda(), self.v.cuda(), self.scale, plan, self.ks.cuda(), self.vs.cuda(),
                        softcap=softcap, slopes=None if slopes is None else slopes.cuda())

    def exact(self, window=0, softcap=0.0, slopes=None):
        return OA.attend(self.q, self.k, self.v, self.ks, self.vs, self.scale, self.starts, self.lens, self.table, softcap, slopes,
                         window, self.prefix, self.shared_table, self.shared_lens, self.of)

    def positions(self):
        return OA.positions(self.starts, self.lens, self.rows, self.shared_lens, self.of)


def check(r, ref, D, what="", softcap=0.0):
    """r: K.attend's dict, ref: oracle.attend.attend's.
    Bounds. A score is a sum of D exact products, each cut at 2^-23 of the largest at worst in the matrix unit, times fp32
    factors (and with a bias one more sum): |ds| <= (D + 8) 2^-23 A with A the row's largest sum of |q_d k_d| (and bias); a cap
    adds 2^-22 of the cap where scores pass an eighth of it, and at most 2^-20 of a score below. A weight is off by its score's
    error, twice (its own and the normaliser's), by 2^-11 where it is rounded to fp16, and by 2^-18 for v_exp_f32, the page's
    factors and the joins; the sums over keys are fp32 sums, 2^-17 of the sum of magnitudes for up to 128 terms in a row.
    fp16 holds nothing finer than 2^-24: a weight p |vs| 2^7 / 2^r is off by 2^-25 where it is below 2^-14, which no relative
    error covers where the heaviest keys hold zeros, and 2^r is at most the largest p |vs| of its pages (page maximum times the
    power of two at or below |vs|): 2^-32 max(p |vs|) of a weight, for each |code| of the sum. So |out - ref| <= (2 ds + 2^-11 +
    2^-16) sum p |v| + 2^-32 max(p |vs|) sum |code| and half a bf16 step, 2^-8 |ref|; |lse - ref| <= ds + 2^-20 (1 + |ref|)."""
    out, lse, mass, reach, grain = ref
    ds = (D + 8) * 2.0 ** -23 * reach + 2.0 ** -22 * softcap + 2.0 ** -20 * reach * bool(softcap)
    got, gl = r["out"].double().cpu(), r["lse"].double().cpu()
    assert got.shape == out.shape and gl.shape == lse.shape
    nan = out.isnan()
    assert torch.equal(got.isnan(), nan), (what, "NaN places", (got.isnan() != nan).sum().item())
    tol = (2 * ds[..., None] + 2.0 ** -11 + 2.0 ** -16) * mass + 2.0 ** -32 * grain + 2.0 ** -8 * out.abs()
    bad = ((got - out).abs() > tol) & ~nan
    assert not bad.any(), (what, "out", (got - out).abs().nan_to_num().max().item(), bad.nonzero()[:4].tolist())
    assert torch.equal(gl.isnan(), lse.isnan()) and torch.equal(gl == -torch.inf, lse == -torch.inf), (what, "lse places")
    fin = lse.isfinite()
    bad = ((gl - lse).abs() > ds + 2.0 ** -20 * (1 + lse.abs()))[fin]
    assert not bad.any(), (what, "lse", (gl - lse)[fin].abs().max().item())
