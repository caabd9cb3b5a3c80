"""A paged batch for the tests, and its operators in 64 bits from their
definitions, a row and a position at a time where that matters."""
import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step


class Batch:
    """`seqs`: (cached positions, new rows) of each sequence. Pages are dealt
    in a shuffled order; `lead` rows before the first sequence's and `tail`
    behind the last are nobody's. layout: "slots" [page][slot][head][d],
    "heads" [page][head][slot][d], "wide" as slots with gaps."""

    def __init__(self, em, heads, kv_heads, head_size, page_size, seqs, dtype="f32", layout="slots",
                 seed=1, lead=0, tail=0, spare_columns=1, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.H, self.KV, self.D, self.ps, self.dtype = heads, kv_heads, head_size, page_size, dtype
        self.seqs = list(seqs)
        need = [-(-(p + r) // page_size) for p, r in seqs]
        self.n_pages = sum(need) + 2
        self.max_pages = max(need + [0]) + spare_columns
        order = torch.randperm(self.n_pages, generator=g)
        self.table = torch.full((len(seqs), self.max_pages), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n].int()
            at += n
        starts = [lead]
        for _, r in seqs:
            starts.append(starts[-1] + r)
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.lengths = torch.tensor([p + r for p, r in seqs], dtype=torch.int32)
        self.rows = starts[-1] + tail
        dt = DTYPES[dtype]
        KV, D, ps, N = kv_heads, head_size, page_size, self.n_pages
        # Cache strides in elements, and the memory they need.
        if layout == "heads":
            self.strides = (KV * ps * D, D, ps * D)
        elif layout == "wide":
            self.strides = (ps * (KV * (D + 8) + 16) + 24, KV * (D + 8) + 16, D + 8)
        else:
            self.strides = (ps * KV * D, KV * D, D)
        size = (N - 1) * self.strides[0] + (ps - 1) * self.strides[1] + (KV - 1) * self.strides[2] + D
        self.kc = torch.randn((size,), generator=g).to(dt)
        self.vc = torch.randn((size,), generator=g).to(dt)
        dim, kv = heads * D, KV * D
        self.qkv = torch.randn((self.rows, dim + 2 * kv), generator=g)
        self.qkv[:, :dim] *= q_scale
        self.shape = em.paged_shape(heads, KV, D, ps, N, self.max_pages, dtype, *self.strides)

    def view(self, cache):
        """[page, slot, head, d] of a cache."""
        return cache.as_strided((self.n_pages, self.ps, self.KV, self.D),
                                (*self.strides[:2], self.strides[2], 1))

    def q(self):
        return self.qkv[:, :self.H * self.D]

    def k(self):
        return self.qkv[:, self.H * self.D:(self.H + self.KV) * self.D]

    def v(self):
        return self.qkv[:, (self.H + self.KV) * self.D:]

    def cuda(self):
        for name in ("table", "starts", "lengths", "kc", "vc", "qkv"):
            setattr(self, name, getattr(self, name).cuda())
        return self

    def batch(self):
        return self.starts, self.lengths, self.table

    # -- definitions ----------------------------------------------------------

    def owner(self, r):
        """(sequence, position) of row r, or (None, None)."""
        st = self.starts.tolist()
        for s in range(len(self.seqs)):
            if st[s] <= r < st[s + 1]:
                return s, int(self.lengths[s]) - (st[s + 1] - r)
        return None, None

    def page(self, s, t):
        """The page of position t of sequence s, or None."""
        if t < 0 or t >= self.max_pages * self.ps:
            return None
        p = int(self.table[s, t // self.ps])
        return p if 0 <= p < self.n_pages else None

    def ref_append(self, freq, halves):
        """(q_out with NaN in rows left alone, key cache, value cache), 64 bits."""
        H, KV, D = self.H, self.KV, self.D
        kc, vc = self.kc.double().cpu(), self.vc.double().cpu()
        kv_, vv = self.view(kc), self.view(vc)
        q_out = torch.full((self.rows, H * D), float("nan"), dtype=torch.float64)
        f = freq.double().cpu()
        n = f.numel()
        i0 = torch.arange(n) * (1 if halves else 2)
        i1 = i0 + (n if halves else 1)

        def rotate(x, pos):
            x = x.double().cpu().clone()
            a = pos * f
            x0, x1 = x[:, i0].clone(), x[:, i1].clone()
            x[:, i0] = x0 * torch.cos(a) - x1 * torch.sin(a)
            x[:, i1] = x0 * torch.sin(a) + x1 * torch.cos(a)
            return x

        for r in range(self.rows):
            s, pos = self.owner(r)
            if s is None or pos < 0 or pos >= self.max_pages * self.ps:
                continue
            q_out[r] = rotate(self.q()[r].reshape(H, D), pos).reshape(-1)
            p = self.page(s, pos)
            if p is not None:
                kv_[p, pos % self.ps] = rotate(self.k()[r].reshape(KV, D), pos)
                vv[p, pos % self.ps] = self.v()[r].reshape(KV, D).double().cpu()
        return q_out, kc, vc

    def ref_attention(self, scale=None, window=0):
        """(out with NaN in rows that are nobody's, tolerance), 64 bits.

        The tolerance: a score is a sum of D products rounded about D times
        with signs of their own, each by at most 2^-24 of S = scale sum |q k|:
        six standard deviations are 6 / sqrt(3) sqrt(D) 2^-24 S. A weight is off by
        that twice (the maximum's too) and by 4 2^-24 for the exponential; the
        sums of n weights and n products are off by 6 / sqrt(3) sqrt(n) 2^-24 of
        them. Times the largest value seen."""
        H, KV, D, G = self.H, self.KV, self.D, self.H // self.KV
        scale = D ** -0.5 if scale is None else scale
        kc, vc = self.view(self.kc.cpu().double()), self.view(self.vc.cpu().double())
        table = self.table.cpu().numpy()
        out = np.full((self.rows, H * D), np.nan)
        tol = np.zeros((self.rows, H * D))
        q_all = self.q().double().cpu().numpy().reshape(self.rows, H, D)
        kn, vn = kc.numpy(), vc.numpy()
        c6 = 6 / np.sqrt(3.0) * 2.0 ** -24
        for r in range(self.rows):
            s, pos = self.owner(r)
            if s is None:
                continue
            first = max(0, pos + 1 - window) if window else 0
            t = np.arange(first, max(first, min(pos + 1, self.max_pages * self.ps)))
            pages = table[s, t // self.ps]
            ok = (pages >= 0) & (pages < self.n_pages)
            t, pages = t[ok], pages[ok]
            if t.size == 0:
                out[r] = 0.0
                continue
            k = kn[pages, t % self.ps]  # (n, KV, D)
            v = vn[pages, t % self.ps]
            for h in range(H):
                kh, vh = k[:, h // G], v[:, h // G]
                with np.errstate(all="ignore"):
                    sc = scale * (kh @ q_all[r, h])
                    w = np.exp(sc - sc.max())
                    out[r, h * D:(h + 1) * D] = (w @ vh) / w.sum()
                    S = abs(scale) * (np.abs(kh) @ np.abs(q_all[r, h]))
                    S = S[np.isfinite(S)].max(initial=0.0)
                    rel = 2 * c6 * np.sqrt(D) * S + 4 * 2.0 ** -24 + 2 * c6 * np.sqrt(t.size)
                    tol[r, h * D:(h + 1) * D] = rel * np.abs(vh).max()
        return out, tol
