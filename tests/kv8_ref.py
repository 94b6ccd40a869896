"""The 8-bit KV cache restated in 64 bits with torch on any device, for the tests: its number format, its records,
attention over the values they hold, and a step's tables as a loop over sequences."""

from __future__ import annotations

import math

import torch

PAGE, DH, REC = 16, 128, 4224


def e4m3_values(device="cpu") -> torch.Tensor:
    """The value of each of the 256 codes (double; NaN for 0x7f and 0xff)."""
    v = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = math.nan if c & 127 == 127 else (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6
        v.append(-x if c & 128 else x)
    return torch.tensor(v, dtype=torch.float64, device=device)


def scale_exp(amax: torch.Tensor) -> torch.Tensor:
    """The scale's exponent of blocks with largest finite magnitudes amax (double)."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = (e.long() - 9 + (m > 0.875).long()).clamp(-100, 118)
    return torch.where(amax == 0, torch.zeros_like(e), e)


def quantise(x: torch.Tensor):
    """x [..., 128] -> (codes int64, scale exponents int64 [...])."""
    x = x.double()
    lut = e4m3_values(x.device)
    fin = torch.isfinite(x)
    e = scale_exp(torch.where(fin, x.abs(), torch.zeros_like(x)).amax(-1))
    y = torch.where(fin, x, torch.zeros_like(x)) * torch.exp2(-e.double())[..., None]
    y = y.clamp(-448, 448)
    mag = lut[:127].contiguous()
    hi = torch.searchsorted(mag, y.abs().contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - mag[lo], mag[hi] - y.abs()
    c = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = c + 128 * torch.signbit(x).long()
    return torch.where(fin, c, torch.full_like(c, 255)), e


def k_at(slot, d):
    return d // 64 * 1024 + d // 16 % 4 * 256 + slot * 16 + d % 16


def v_at(slot, d):
    return 2048 + d // 64 * 1024 + slot // 4 * 256 + d % 16 * 16 + d // 16 % 4 * 4 + slot % 4


def scales(pool: torch.Tensor) -> torch.Tensor:
    """The scales of a pool, fp32 [pages, Hkv, 32] (a view)."""
    return pool[..., 4096:].view(torch.float32)


def write(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots) -> None:
    """k, v [B, Hkv, 128] into the pool's records at slots (those outside the pool left out)."""
    d = torch.arange(DH, device=pool.device)
    (kc, ke), (vc, ve) = quantise(k), quantise(v)
    sc = scales(pool)
    for b, s in enumerate(torch.as_tensor(slots).tolist()):
        if not 0 <= s < pool.shape[0] * PAGE:
            continue
        p, t = divmod(s, PAGE)
        pool[p][:, k_at(t, d)] = kc[b].to(torch.uint8)
        pool[p][:, v_at(t, d)] = vc[b].to(torch.uint8)
        sc[p, :, t] = torch.exp2(ke[b].double()).float()
        sc[p, :, PAGE + t] = torch.exp2(ve[b].double()).float()


def read(pool: torch.Tensor, pages) -> tuple:
    """k, v (double [Hkv, 16 n, 128]) that the given pages hold."""
    dev = pool.device
    rec = pool[torch.as_tensor(pages, device=dev).long()]
    lut, d, t = e4m3_values(dev), torch.arange(DH, device=dev), torch.arange(PAGE, device=dev)
    sc = scales(rec).double()
    out = []
    for at, s in ((k_at(t[:, None], d[None]), sc[..., :PAGE]), (v_at(t[:, None], d[None]), sc[..., PAGE:])):
        x = lut[rec[..., at.reshape(-1)].long()].view(*rec.shape[:2], PAGE, DH) * s[..., None]
        out.append(x.permute(1, 0, 2, 3).reshape(rec.shape[1], -1, DH))
    return tuple(out)


def random_pool(pages: int, Hkv: int, seed: int, device="cpu", v_spread: float = 0.7) -> torch.Tensor:
    """A pool full of normal keys and values of uneven tokens."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((pages * PAGE, Hkv, DH), generator=g, dtype=torch.float64)
    v = torch.randn((pages * PAGE, Hkv, DH), generator=g, dtype=torch.float64)
    v = v * torch.exp(v_spread * torch.randn((pages * PAGE, Hkv, 1), generator=g, dtype=torch.float64))
    (kc, ke), (vc, ve) = quantise(k), quantise(v)
    kc, vc = (c.to(torch.uint8).view(pages, PAGE, Hkv, DH) for c in (kc, vc))
    pool = torch.zeros((pages, Hkv, REC), dtype=torch.uint8)
    d = torch.arange(DH)
    sc = scales(pool)
    for t in range(PAGE):
        pool[:, :, k_at(t, d)] = kc[:, t]
        pool[:, :, v_at(t, d)] = vc[:, t]
        sc[:, :, t] = torch.exp2(ke.double()).float().view(pages, PAGE, Hkv)[:, t]
        sc[:, :, PAGE + t] = torch.exp2(ve.double()).float().view(pages, PAGE, Hkv)[:, t]
    return pool.to(device)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, keep: torch.Tensor | None = None):
    """(out, tol) of q [n, G, 128] rows over one kv head's k, v [N, 128] (double), where keep [n, N] says which keys
    each row sees; rows that see none give zeros.  tol is how far the kernels' bf16 outputs may be off:
      * half a bf16 step of the output, 2^-8 |out|;
      * against sum p |v| = A: half an fp16 step of each probability, 2^-11; the fp32 sums, one rounding of 2^-24 a
        32-key step on either side of the division; scores off by 2^-24 for each of 128 products and the scale,
        times sum |q||k| scale, doubled since numerator and denominator both move; exp2 and divisions, 2^-20;
      * probabilities below fp16's range (2^-40 of the largest) and values 2^32 below the loudest, absolute."""
    q = q.double()
    s = torch.einsum("ngd,kd->ngk", q, k) * scale
    mag = torch.einsum("ngd,kd->ngk", q.abs(), torch.nan_to_num(k).abs()) * scale
    if keep is not None:
        s = s.masked_fill(~keep[:, None, :], -math.inf)
        mag = mag.masked_fill(~keep[:, None, :], 0.0)
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:2], 1), -math.inf)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l, torch.zeros_like(p))
    seen = torch.ones(k.shape[0], dtype=torch.bool, device=k.device) if keep is None else keep.any(0)
    vs = torch.where(seen[:, None], v, torch.zeros_like(v))
    out = torch.einsum("ngk,kd->ngd", p, vs)
    A = torch.einsum("ngk,kd->ngd", p, vs.abs())
    n, vmax = k.shape[0], float(vs.abs().amax()) if vs.numel() else 0.0
    ds = mag.amax(-1, keepdim=True) * 130 * 2.0 ** -24 if s.shape[-1] else 0.0
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -11 + (n / 32 + 8) * 2.0 ** -23 + 2 * ds + 2.0 ** -20) * A
    return out, tol + vmax * (n * 2.0 ** -40 + 2.0 ** -31) + 2.0 ** -133


def step_tables(ctx, new, table, rows: int, free=None, free_at: int = 0) -> dict:
    """jit_step_tables as a loop; `table` (a list of lists) grows in place.  Sums past int32 stay at its largest."""
    top = 2 ** 31 - 1
    W = len(table[0]) if table else 1
    out = {"row_start": [0], "row_seq": [-1] * rows, "pos": [0] * rows, "slots": [-1] * rows, "lens": []}
    at, nxt, refused, end = free_at, free_at, 0, 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        start, end = end, end + n
        have, tot = -(-c // PAGE), -(-(c + n) // PAGE)
        fits = tot <= W and end <= rows
        need = tot - have if fits and free is not None else 0
        at += need
        served = fits and (need == 0 or at <= len(free))
        if served and need:
            table[b][have:tot] = free[at - need:at]
            nxt = at
        refused += not served
        for i in range(min(n, max(0, rows - start))):
            if start + i < rows:
                out["row_seq"][start + i], out["pos"][start + i] = b, min(c + i, top)
                page = table[b][(c + i) // PAGE] if served else -1
                out["slots"][start + i] = page * PAGE + (c + i) % PAGE if 0 <= page < 1 << 27 else -1
        out["row_start"].append(min(end, top))
        out["lens"].append(min(c + n, top) if served else c)
    out["status"] = [min(end, top), nxt, refused, 0]
    return out
