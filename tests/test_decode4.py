"""The operators of a decode layer in 4 bits: ling_b200_nvfp4_matvec, ling_b200_kv4_append / _read / _attention.

On the GPU each is held to its formula in 64 bits.  Tolerances count roundings (a value rounded to t is off by at most
finfo(t).eps / 2 of itself) and bound the fp32 sums by their absolute terms:
  matvec     eps(y)/2 |y| + 2^-23 (K/16 + 64) sum |x w| alpha      (at most K/16 + 64 dependent additions of a tensor-core sum)
  rotation   eps/2 |q'| + 2^-22 (|x cos| + |o sin|)
  codes      none: the cache holds exactly what the formula gives
  attention  eps/2 |o| + (2^-11 + 2 E + 2^-19) sum p|v| / sum p + 2^-33 sum |v| / sum p, E = 2^-23 (D + 8) max scale sum |q||k|: the
             probabilities may be rounded to FP16 for the tensor cores, and a score's error E moves a probability by E of
             itself, above and below the fraction.  FP16 steps do not shrink below 2^-24, so a small probability (the largest is 1, carried
             times 2^8) is off by up to 2^-25 / 2^8 = 2^-33 whatever its size, which the last term counts over the visible keys.
Refusals are checked without a GPU: every argument is looked at before the device is."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAG = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BAD_PAGE, BAD_BATCH = 5, 8


# ------------------------------------------------------------------------------------------------ 64-bit forms
def e4m3_table():
    out = []
    for b in range(256):
        e, f = b >> 3 & 15, b & 7
        v = math.nan if b & 127 == 127 else f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        out.append(-v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def values64(codes, scales):
    dev = codes.device
    mag = torch.tensor(MAG + [-m for m in MAG], dtype=torch.float64, device=dev)
    x = mag[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return x * e4m3_table().to(dev)[scales.long()].repeat_interleave(16, -1)


def stored64(x):
    """What a cache holds of the vectors x (float64 [.., D], tensor scale taken off): the formula, from tables."""
    if x.numel() == 0:
        return x
    g = x.unflatten(-1, (-1, 16))
    tab = e4m3_table()[:127].to(x.device)
    # the scale is the E4M3 value nearest the fp32 quotient amax / 6, halfway to the even code
    want = (torch.nan_to_num(g, 0, 0, 0).abs().amax(-1) / 6).clamp(2.0 ** -9, 448).float().double()
    hi = torch.searchsorted(tab, want).clamp(1, 126)
    lo = hi - 1
    d = (want - tab[lo]) - (tab[hi] - want)
    sc = tab[torch.where((d > 0) | ((d == 0) & (hi % 2 == 0)), hi, lo)].unsqueeze(-1)
    mag = torch.tensor(MAG, dtype=torch.float64, device=x.device)
    border = (mag[1:] + mag[:-1]) / 2
    code = (g.abs().unsqueeze(-1) > border * sc.unsqueeze(-1)).sum(-1)  # halfway: the smaller magnitude
    out = (torch.where(g < 0, -1.0, 1.0) * mag[code] * sc).flatten(-2)
    return torch.where((~torch.isfinite(x)).any(-1, keepdim=True), math.nan, out)


def rotated64(x, p, rot, theta):
    x = x.double()
    h = rot // 2
    if h == 0:
        return x
    a = p.double()[:, None, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device), torch.arange(h, device=x.device, dtype=torch.float64) * (-2.0 / rot))
    lo, hi = x[..., :h], x[..., h:rot]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), x[..., rot:]], -1)


def random_nvfp4(shape, gen, spread=1.0):
    x = torch.randn(shape, device="cuda", generator=gen) * spread
    g = x.reshape(*shape[:-1], -1, 16)
    s = (g.abs().amax(-1) / 6).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
    c = torch.bucketize(g.abs() / s.float().unsqueeze(-1), torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.], device="cuda")).to(torch.uint8) + 8 * (g < 0).to(torch.uint8)
    c = c.reshape(*shape[:-1], -1, 2)
    return (c[..., 0] | c[..., 1] << 4).contiguous(), s.view(torch.uint8).contiguous()


# ------------------------------------------------------------------------------------------------ refusals, without a GPU
def _p(n=1):
    return C.c_void_p(4096 * n)  # never dereferenced


def c_cache(lb, **kw):
    a = dict(k=4096, v=8192, k_scales=16384, v_scales=32768, tables=65536, kv_heads=2, head_dim=128, page_tokens=16, pages=8, slots=2, max_pages=4,
             k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return lb._Kv4(**a)


def c_batch(lb, **kw):
    a = dict(row0=4096, slot=8192, pos=16384, rope_pos=None, anc=None, seqs=2, rows=8, max_rows=4, max_context=64)
    a.update(kw)
    return lb._Kv4Batch(**a)


@pytest.mark.parametrize("change", [dict(M=0), dict(M=33), dict(K=24), dict(K=0), dict(N=0), dict(ldx=31), dict(ldy=7), dict(xt=3), dict(yt=-1), dict(x=None),
                                    dict(w=None), dict(ws=None), dict(y=None), dict(x=C.c_void_p(4097)), dict(y=C.c_void_p(4098)), dict(w=C.c_void_p(4100)), dict(device=-1)])
def test_matvec_refusals(lb, change):
    a = dict(device=0, x=_p(), xt=lb.BF16, ldx=32, M=1, w=_p(2), ws=_p(3), N=8, K=32, y=_p(4), yt=lb.F32, ldy=8)
    a.update(change)
    fn = lb.lib().ling_b200_nvfp4_matvec
    fn.argtypes = lb._MATVEC_ARGS
    assert fn(a["device"], a["x"], a["xt"], a["ldx"], a["M"], a["w"], a["ws"], 1.0, a["N"], a["K"], a["y"], a["yt"], a["ldy"], 0, None) == lb.ERR_ARG
    assert lb.last_error()


def calls(lb, cache, batch, rows=(4096, 256, 128), type_=1, q_heads=4, rot=64, theta=1e7, scale=0.1, ws=1 << 40, out=(8192, 512, 128), wsp=4096, q=(4096, 512, 128)):
    L, b = lb.lib(), C.byref
    c, bt, kv, o, qr = cache, batch, lb._Rows(*rows), lb._Rows(*out), lb._Rows(*q)
    L.ling_b200_kv4_attention_workspace.restype = C.c_size_t
    L.ling_b200_kv4_append.argtypes = L.ling_b200_kv4_read.argtypes = L.ling_b200_kv4_attention.argtypes = None
    return (L.ling_b200_kv4_append(0, b(c), b(bt), type_, b(kv), b(kv), b(qr), q_heads, b(o), rot, C.c_double(theta), None, None),
            L.ling_b200_kv4_read(0, b(c), b(bt), type_, b(kv), b(kv), None, None),
            L.ling_b200_kv4_attention(0, b(c), b(bt), type_, b(qr), q_heads, C.c_float(scale), b(o), None, C.c_void_p(wsp), C.c_size_t(ws), None, None))


@pytest.mark.parametrize("change", [dict(k=0), dict(tables=0), dict(k=4100), dict(v_scales=32770), dict(head_dim=96), dict(page_tokens=48), dict(page_tokens=8),
                                    dict(kv_heads=0), dict(pages=0), dict(slots=0), dict(max_pages=0), dict(k_scale=0.3), dict(v_scale=0.0), dict(k_scale=math.nan),
                                    dict(v_scale=2.0 ** 31), dict(pages=1 << 27), dict(pages=(1 << 31) - 1)])
def test_cache_refusals(lb, change):
    assert calls(lb, c_cache(lb, **change), c_batch(lb)) == (lb.ERR_ARG,) * 3 and lb.last_error()


@pytest.mark.parametrize("change", [dict(row0=0), dict(slot=0), dict(pos=0), dict(pos=4097), dict(anc=3), dict(seqs=0), dict(seqs=1025), dict(rows=-1), dict(max_rows=9),
                                    dict(max_rows=-1), dict(max_context=3), dict(max_context=65), dict(rows=64, max_rows=33, anc=4096)])
def test_batch_refusals(lb, change):
    assert calls(lb, c_cache(lb), c_batch(lb, **change)) == (lb.ERR_ARG,) * 3 and lb.last_error()


def test_other_refusals(lb):
    ok = c_cache(lb), c_batch(lb)
    assert calls(lb, *ok, type_=3) == (lb.ERR_ARG,) * 3
    assert calls(lb, *ok, rows=(4097, 256, 128), q=(4097, 512, 128)) == (lb.ERR_ARG,) * 3
    assert calls(lb, *ok, rows=(4096, 64, 128), q=(4096, 64, 128)) == (lb.ERR_ARG,) * 3
    assert calls(lb, *ok, rot=3)[0] == lb.ERR_ARG and calls(lb, *ok, rot=130)[0] == lb.ERR_ARG
    assert calls(lb, *ok, theta=0.0)[0] == lb.ERR_ARG and calls(lb, *ok, theta=math.inf)[0] == lb.ERR_ARG
    assert calls(lb, *ok, type_=0)[2] == lb.ERR_ARG                       # fp32 queries
    assert calls(lb, *ok, q_heads=3)[2] == lb.ERR_ARG                     # not a multiple of the kv heads
    assert calls(lb, *ok, scale=math.nan)[2] == lb.ERR_ARG
    assert calls(lb, *ok, ws=8)[2] == lb.ERR_ARG and calls(lb, *ok, wsp=0)[2] == lb.ERR_ARG and calls(lb, *ok, wsp=4104)[2] == lb.ERR_ARG
    assert calls(lb, *ok, out=(8192, 256, 128)) [0] == lb.ERR_ARG         # rows of the output overlap
    assert "overlap" in lb.last_error()
    assert lb.lib().ling_b200_kv4_attention_workspace(C.byref(ok[0]), C.byref(ok[1]), 3) == 0
    # an empty call is a call: nothing is launched, no device is needed
    assert calls(lb, c_cache(lb), c_batch(lb, rows=0, max_rows=0)) == (lb.OK,) * 3
    assert calls(lb, c_cache(lb), c_batch(lb, rows=0, max_rows=0), rows=(0, 256, 128), q=(0, 512, 128), out=(0, 512, 128), wsp=0) == (lb.OK,) * 3


def test_host_arrays_are_refused(lb):
    z = torch.zeros(4, 4)
    with pytest.raises(lb.LingError):
        lb.nvfp4_matvec(z, torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 1.0, z)
    with pytest.raises(lb.LingError):
        lb.Kv4Batch(z.int(), z.int(), z.int(), 1, 1, 1)
    with pytest.raises(lb.LingError):
        lb.Kv4Cache(z, z, z, z, z)


# ------------------------------------------------------------------------------------------------ matvec
def matvec_case(lb, M, N, K, xt, yt, seed=0, accumulate=False, x_off=0, w_off=0, ldx=None, ldy=None, spread=2.0):
    gen = torch.Generator("cuda").manual_seed(seed + 1000 * M + N + K)
    w, ws = random_nvfp4((N, K), gen, spread)
    if w_off:  # values that start off an 8-byte boundary
        flat = torch.zeros(w.numel() + w_off, dtype=torch.uint8, device="cuda")
        flat[w_off:] = w.flatten()
        w = flat[w_off:].view(N, K // 2)
    buf = torch.randn(M, (ldx or K) + x_off, device="cuda", generator=gen).to(T[xt])
    x = buf[:, x_off:x_off + K]
    y = torch.full((M, ldy or N), 3.0, dtype=T[yt], device="cuda")[:, :N]
    y0 = y.double()
    lb.nvfp4_matvec(x, w, ws, 0.37, y, accumulate=accumulate)
    w64, x64 = values64(w, ws), x.double()
    want = 0.37 * x64 @ w64.t() + (y0 if accumulate else 0)
    alpha = float(np.float32(0.37))
    want = alpha * (x64 @ w64.t()) + (y0 if accumulate else 0)
    terms = alpha * (x64.abs() @ w64.abs().t())
    tol = torch.finfo(T[yt]).eps / 2 * want.abs() + 2.0 ** -23 * (K / 16 + 64) * terms + 2.0 ** -22 * (y0.abs() if accumulate else 0) + 2.0 ** -24 * (T[yt] == torch.float16)
    assert torch.isfinite(y.double()).all()
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max().item()
    return x, w, ws, y


@pytest.mark.gpu
@pytest.mark.parametrize("xt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 1024, 5120), (2, 7, 48), (3, 33, 1008), (8, 129, 272), (9, 64, 4096), (16, 1000, 528), (17, 250, 2064), (32, 515, 1296)])
def test_matvec(gpu, lb, M, N, K, xt):
    for yt in ("bf16", "f16", "f32"):
        matvec_case(lb, M, N, K, xt, yt)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(accumulate=True), dict(x_off=1), dict(x_off=8), dict(ldx=1111), dict(w_off=8), dict(w_off=24), dict(ldy=77), dict(accumulate=True, yt="f16"),
                                dict(xt="f32", x_off=3, ldx=1200), dict(xt="f32", accumulate=True, yt="bf16")])
def test_matvec_strides_and_alignment(gpu, lb, kw):
    kw = dict(kw)
    for M in (1, 5, 20):
        matvec_case(lb, M, 75, 1088, kw.get("xt", "bf16"), kw.get("yt", "f32"), **{k: v for k, v in kw.items() if k not in ("xt", "yt")})


@pytest.mark.gpu
@pytest.mark.parametrize("xt", ["bf16", "f16", "f32"])
def test_matvec_rows_are_independent_and_calls_repeat(gpu, lb, xt):
    x, w, ws, y = matvec_case(lb, 32, 300, 2560, xt, "f32")
    again = torch.zeros_like(y)
    lb.nvfp4_matvec(x, w, ws, 0.37, again)
    assert torch.equal(again, y)
    for m in (0, 13, 31):
        one = torch.zeros(1, 300, device="cuda")
        lb.nvfp4_matvec(x[m:m + 1], w, ws, 0.37, one)
        assert torch.allclose(one, y[m:m + 1], rtol=0, atol=float(2.0 ** -22 * (2560 / 16 + 64) * 0.37 * (x[m].double().abs() @ values64(w, ws).abs().t()).max()))
    bad = x.clone()
    bad[5, 100] = math.nan
    out = torch.zeros_like(y)
    lb.nvfp4_matvec(bad, w, ws, 0.37, out)
    assert torch.isnan(out[5]).all() and torch.equal(out[:5], y[:5]) and torch.equal(out[6:], y[6:])


@pytest.mark.gpu
def test_matvec_wide_values_of_f32_rows(gpu, lb):
    """fp32 rows whose magnitudes span 2^-40 .. 2^40 keep fp32's precision."""
    gen = torch.Generator("cuda").manual_seed(5)
    w, ws = random_nvfp4((64, 512), gen)
    x = torch.randn(3, 512, device="cuda", generator=gen) * torch.exp2(torch.randint(-40, 41, (3, 512), device="cuda", generator=gen).float())
    y = torch.zeros(3, 64, device="cuda")
    lb.nvfp4_matvec(x, w, ws, 1.0, y)
    w64 = values64(w, ws)
    assert ((y.double() - x.double() @ w64.t()).abs() <= 2.0 ** -23 * (512 / 16 + 64) * (x.double().abs() @ w64.abs().t())).all()


# ------------------------------------------------------------------------------------------------ the cache
class Setup:
    """A cache with shuffled pages for sequences of (rows, positions already there)."""

    def __init__(self, lb, seqs, D, H, page, seed=0, fill=None, tree=False, padded=0, slack=0, extra_slots=1):
        gen = torch.Generator("cuda").manual_seed(seed)
        n = len(seqs)
        need = [max(1, -(-(r + p) // page)) for r, p in seqs]
        self.pages, most, slots = sum(need) + 3, max(need) + 1, n + extra_slots
        perm = (torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)) + 1).int()
        slot = torch.randperm(slots, generator=torch.Generator().manual_seed(seed + 1))[:n].int()
        tables = torch.zeros(slots, most, dtype=torch.int32)
        at = 0
        for s in range(n):
            tables[slot[s], :need[s]] = perm[at:at + need[s]]
            at += need[s]
        self.tables, self.slot = tables.cuda(), slot.cuda()
        rows = [r for r, _ in seqs]
        self.total = sum(rows)
        self.rows = self.total + padded
        self.row0 = torch.tensor([sum(rows[:i]) for i in range(n + 1)], dtype=torch.int32).cuda()
        self.pos = torch.tensor([p for _, p in seqs], dtype=torch.int32).cuda()
        self.seqs, self.D, self.H, self.page, self.gen = seqs, D, H, page, gen
        shape = (self.pages + 1, H, page, D)
        if fill is None:
            (self.k, self.ks), (self.v, self.vs) = random_nvfp4(shape, gen), random_nvfp4(shape, gen)
        else:
            self.k, self.v = (torch.full((*shape[:3], D // 2), fill, dtype=torch.uint8, device="cuda") for _ in range(2))
            self.ks, self.vs = (torch.full((*shape[:3], D // 16), fill, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.anc = None
        if tree:
            m = []
            for r in rows:
                mine = []
                for i in range(r):
                    parent = -1 if i == 0 else int(torch.randint(0, i, (1,), generator=torch.Generator().manual_seed(seed + i)))
                    mine.append((mine[parent] if parent >= 0 else 0) | 1 << i)
                m += mine
            self.masks = m + [0] * padded
            self.anc = torch.tensor([x - (1 << 32) if x >> 31 else x for x in self.masks], dtype=torch.int32).cuda()
        self.max_rows, self.max_context = max(rows), max(r + p for r, p in seqs) + slack
        self.of = torch.cat([torch.full((r,), s) for s, (r, _) in enumerate(seqs)]).long().cuda() if self.total else torch.zeros(0, dtype=torch.long, device="cuda")
        self.at = torch.cat([torch.arange(r) + p for r, p in seqs]).long().cuda()
        self.lb = lb

    def batch(self, **kw):
        return self.lb.Kv4Batch(self.row0, self.slot, self.pos, self.rows, self.max_rows, self.max_context, anc=self.anc, **kw)

    def cache(self, **kw):
        return self.lb.Kv4Cache(self.k, self.ks, self.v, self.vs, self.tables, **kw)

    def where(self, s, p):
        """Pages and tokens of positions p of sequence s."""
        return self.tables[self.slot[s].long(), p // self.page].long(), p % self.page

    def held(self, s, n):
        p = torch.arange(n, device="cuda")
        page, tok = self.where(s, p)
        return values64(self.k[page, :, tok], self.ks[page, :, tok]), values64(self.v[page, :, tok], self.vs[page, :, tok])  # [n][H][D]

    def visible(self, s):
        """[rows of s][positions]"""
        r, p = self.seqs[s]
        j = torch.arange(r + p, device="cuda") - p
        if self.anc is None:
            return j[None] <= torch.arange(r, device="cuda")[:, None]
        m = torch.tensor(self.masks[int(self.row0[s]):int(self.row0[s]) + r], device="cuda", dtype=torch.long)
        return (j < 0)[None] | ((m[:, None] >> j.clamp(0, 31)[None]) & 1 == 1) & (j >= 0)[None]


def check_append(lb, s, t, q_heads, rot, rope=None, theta=1e6, k_scale=1.0, v_scale=1.0, poke=None, layout="apart"):
    D, H, R = s.D, s.H, s.rows
    if layout == "slice":  # q | k | v of one projection's rows, and one column in front
        buf = torch.randn(R, (q_heads + 2 * H) * D + 8, device="cuda", generator=s.gen).to(T[t])[:, 8:].unflatten(1, (-1, D))
        q, k, v = buf[:, :q_heads], buf[:, q_heads:q_heads + H], buf[:, q_heads + H:]
    elif layout == "odd":  # off every vector boundary
        q, k, v = (torch.randn(R, h * D + 3, device="cuda", generator=s.gen).to(T[t])[:, 1:1 + h * D].unflatten(1, (-1, D)) for h in (max(q_heads, 1), H, H))
    else:  # head-major
        q, k, v = (torch.randn(h, R, D, device="cuda", generator=s.gen).to(T[t]).transpose(0, 1) for h in (max(q_heads, 1), H, H))
    if poke:
        poke(k, v)
    q = q if q_heads else None
    q_out = torch.full((R, q_heads, D), 9.0, dtype=T[t], device="cuda") if q_heads else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = [x.clone() for x in (s.k, s.ks, s.v, s.vs)]
    batch, cache = s.batch(rope_pos=rope), s.cache(k_scale=k_scale, v_scale=v_scale)
    cache.append(batch, k, v, q=q, q_out=q_out, rotary_dim=rot, theta=theta, err=err)
    assert err.item() == 0
    n, rp = s.total, (s.at if rope is None else rope[:s.total].long())
    want_k = stored64(rotated64(k[:n], rp, rot, theta) / k_scale) * k_scale
    want_v = stored64(v[:n].double() / v_scale) * v_scale
    page, tok = s.tables[s.slot[s.of].long(), s.at // s.page].long(), s.at % s.page
    got_k, got_v = values64(s.k[page, :, tok], s.ks[page, :, tok]) * k_scale, values64(s.v[page, :, tok], s.vs[page, :, tok]) * v_scale
    assert torch.equal(got_k.nan_to_num(77), want_k.nan_to_num(77)) and torch.equal(got_v.nan_to_num(77), want_v.nan_to_num(77))
    touched = torch.zeros(s.k.shape[:3], dtype=torch.bool, device="cuda")
    touched[page, :, tok] = True
    for was, now in zip(before, (s.k, s.ks, s.v, s.vs)):  # nothing else was written
        assert torch.equal(was[~touched], now[~touched])
    if q_heads:
        want = rotated64(q[:n], rp, rot, theta)
        size = rotated64(q[:n].double().abs(), rp * 0, 0, theta)
        other = torch.cat([size[..., rot // 2:rot], size[..., :rot // 2], size[..., rot:]], -1)
        assert ((q_out[:n].double() - want).abs() <= torch.finfo(T[t]).eps / 2 * want.abs() + 2.0 ** -22 * (size + other) + 2.0 ** -24 * (t == "f16")).all()
        assert (q_out[n:] == 9.0).all()
        if layout == "slice":  # in place
            inplace = q.clone()
            cache.append(batch, k, v, q=inplace, q_out=inplace, rotary_dim=rot, theta=theta)
            assert torch.equal(inplace[:n], q_out[:n]) and torch.equal(inplace[n:], q[n:])
    for rt in ("bf16", "f32"):
        ko, vo = (torch.full((R, H, D), 9.0, dtype=T[rt], device="cuda") for _ in range(2))
        cache.read(batch, ko, vo, err=err)
        assert err.item() == 0 and (ko[n:] == 9.0).all() and (vo[n:] == 9.0).all()
        assert torch.equal(ko[:n].double().nan_to_num(77), got_k.nan_to_num(77)) and torch.equal(vo[:n].double().nan_to_num(77), got_v.nan_to_num(77))


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,H,q_heads,rot,page,layout", [(64, 1, 0, 64, 16, "apart"), (64, 3, 6, 16, 32, "odd"), (128, 2, 8, 128, 64, "slice"), (128, 5, 5, 0, 16, "slice"),
                                                         (256, 4, 24, 64, 16, "apart"), (256, 1, 3, 256, 128, "odd"), (128, 2, 2, 6, 16, "slice")])
def test_append(gpu, lb, D, H, q_heads, rot, page, layout, t):
    s = Setup(lb, [(3, 14), (0, 5), (1, 0), (20, 100), (70, 31)], D, H, page, seed=D + H, fill=0xff, padded=2)
    check_append(lb, s, t, q_heads, rot, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,q_heads,rot,layout,t", [(64, 2, 3, 32, "slice", "bf16"), (64, 2, 3, 36, "apart", "f32"), (128, 1, 5, 20, "slice", "f16"), (256, 1, 2, 256, "odd", "bf16"),
                                                      (128, 1, 1, 0, "apart", "bf16")])
def test_append_many_rows(gpu, lb, D, H, q_heads, rot, layout, t):
    """Several rows a block: blocks that cross from one sequence to the next, and into the padding."""
    s = Setup(lb, [(1201, 5), (0, 3), (2500, 700), (1, 77), (6, 0), (1003, 16)], D, H, 16, seed=rot, fill=0x33, padded=13)
    check_append(lb, s, t, q_heads, rot, layout=layout)


@pytest.mark.gpu
def test_append_one_token_many_sequences_far_positions(gpu, lb):
    s = Setup(lb, [(1, 37 * i) for i in range(70)] + [(1, 131071)], 128, 2, 64, seed=3, fill=0)
    rope = torch.randint(0, 1 << 24, (s.rows,), device="cuda", generator=s.gen).int()
    check_append(lb, s, "bf16", 4, 128, rope=rope, theta=1e7)


@pytest.mark.gpu
def test_append_values_on_borders_zeros_and_tensor_scales(gpu, lb):
    """Exact halfway values, zero vectors, values below and above every scale, at position 0 (the rotation is the identity)."""
    for ks, vs in ((1.0, 1.0), (2.0 ** -7, 2.0 ** 5)):
        def poke(k, v):
            for x, sc in ((k, ks), (v, vs)):
                x[0, 0] = 0
                steps = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, 0.], device="cuda")
                for e, i in zip((1.0, 1.125, 0.40625, 2.0 ** -9), range(4)):
                    x[0, 1, 16 * i:16 * i + 16] = (steps * (e * sc)).to(x.dtype)
                x[1, 0] = 1e-6 * sc
                x[1, 1] = 5000.0 * sc
                x[2, 0, 16:32] = -2689.0 * sc
        s = Setup(lb, [(1, 0), (1, 0), (1, 0), (1, 0)], 64, 2, 16, seed=9, fill=0x55)
        check_append(lb, s, "bf16", 0, 64, k_scale=ks, v_scale=vs, poke=poke)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_append_vectors_that_are_not_finite_are_nan_whole(gpu, lb, t):
    def poke(k, v):
        k[0, 0, 3], k[1, 1, 127], v[2, 0, 64], v[3, 1, 0] = math.nan, math.inf, -math.inf, math.nan
    check_append(lb, Setup(lb, [(4, 10), (2, 3)], 128, 2, 16, seed=4, fill=1), t, 2, 32, poke=poke)


@pytest.mark.gpu
def test_append_and_read_skip_and_record_what_is_out_of_bounds(gpu, lb):
    for what, code in (("page 0", BAD_PAGE), ("page past the pool", BAD_PAGE), ("slot", BAD_BATCH), ("position", BAD_BATCH), ("rows", BAD_BATCH)):
        s = Setup(lb, [(2, 14), (3, 30)], 64, 1, 16, fill=0x11)
        if what == "page 0":
            s.tables[s.slot[1].long(), 2] = 0
        elif what == "page past the pool":
            s.tables[s.slot[1].long(), 2] = s.pages + 1
        elif what == "slot":
            s.slot[1] = s.tables.shape[0]
        elif what == "position":
            s.pos[1] = s.max_context - 2
        else:
            s.max_rows = 2
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        k = torch.randn(5, 1, 64, device="cuda", generator=s.gen)
        out = torch.full((5, 1, 64), 9.0, device="cuda")
        s.cache().append(s.batch(), k, k, err=err)
        assert err.item() == code, what
        err.zero_()
        s.cache().read(s.batch(), out, None, err=err)
        assert err.item() == code and torch.equal(out[:2].double(), stored64(k[:2].double()))
        kept = out[2:4] if code == BAD_PAGE else None  # positions 30, 31 are on a good page, 32 is not
        assert (kept is None or torch.equal(kept.double(), stored64(k[2:4].double()))) and (out[4:] == 9.0).all()
        assert (s.k[0] == 0x11).all()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(lb, s, t, G, scale=None, spread=1.0, layout="apart", k_scale=1.0, v_scale=1.0, lse=True, q=None, err_code=0, work=None, skip=None):
    D, H, R = s.D, s.H, s.rows
    Q = H * G
    scale = 1 / math.sqrt(D) if scale is None else scale
    if q is None:
        q = torch.randn(R, Q, D, device="cuda", generator=s.gen) * spread
    if layout == "slice":
        q = torch.cat([torch.zeros(R, 8, device="cuda"), q.flatten(1), torch.zeros(R, 8, device="cuda")], 1).to(T[t])[:, 8:8 + Q * D].unflatten(1, (Q, D))
        out = torch.full((R, Q * D + 16), 9.0, dtype=T[t], device="cuda")[:, 8:8 + Q * D].unflatten(1, (Q, D))
    elif layout == "odd":
        q = torch.cat([torch.zeros(R, 1, device="cuda"), q.flatten(1), torch.zeros(R, 2, device="cuda")], 1).to(T[t])[:, 1:1 + Q * D].unflatten(1, (Q, D))
        out = torch.full((R, Q * D + 3), 9.0, dtype=T[t], device="cuda")[:, 1:1 + Q * D].unflatten(1, (Q, D))
    else:
        q = q.to(T[t]).transpose(0, 1).contiguous().transpose(0, 1)
        out = torch.full((Q, R, D), 9.0, dtype=T[t], device="cuda").transpose(0, 1)
    L = torch.full((R, Q), 9.0, device="cuda") if lse else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache, batch = s.cache(k_scale=k_scale, v_scale=v_scale), s.batch()
    if work is None:
        work = torch.zeros(cache.attention_workspace_bytes(batch, Q), dtype=torch.uint8, device="cuda")
    cache.attention(batch, q, out, scale, work, lse=L, err=err)
    assert err.item() == err_code
    scale = float(np.float32(scale))
    for i, (r, p) in enumerate(s.seqs):
        a = int(s.row0[i])
        if r == 0 or (skip and i in skip):
            continue
        k, v = s.held(i, r + p)
        k, v = k * k_scale, v * v_scale
        see = s.visible(i)
        for h in range(Q):
            kh, vh, qh = k[:, h // G], v[:, h // G], q[a:a + r, h].double()
            sc = (scale * (qh @ kh.t())).masked_fill(~see, -math.inf)
            m = sc.amax(-1, keepdim=True)
            e = torch.where(see, (sc - m.nan_to_num(0, neginf=0)).exp(), 0.0)
            l = e.sum(-1, keepdim=True)
            o = (e @ vh.nan_to_num(0)) / l
            o = torch.where((see & torch.isnan(vh).any(-1)).any(-1, keepdim=True), math.nan, o)  # a NaN vector is NaN whole
            o = torch.where(see.any(-1, keepdim=True), o, 0.0)
            A = (e @ vh.abs().nan_to_num(0)) / l.clamp(min=1e-300)
            tail = (see.double() @ vh.abs().nan_to_num(0)) / l.clamp(min=1.0)
            E = 2.0 ** -23 * (D + 8) * abs(scale) * (qh.abs() @ kh.abs().nan_to_num(0).t()).amax(-1, keepdim=True)
            tol = torch.finfo(T[t]).eps / 2 * o.abs() + (2.0 ** -11 + 2 * E + 2.0 ** -19) * A + 2.0 ** -33 * tail + 2.0 ** -24 * (t == "f16")
            got = out[a:a + r, h].double()
            assert torch.equal(torch.isnan(got), torch.isnan(o)), (i, h)
            bad = ((got - o).abs() > tol) & ~torch.isnan(o)
            assert not bad.any(), (i, h, ((got - o).abs() / tol).nan_to_num(0).max().item())
            if lse:
                want = torch.where(see.any(-1), (m + l.log()).squeeze(-1), -math.inf)
                g = L[a:a + r, h].double()
                ok = torch.isnan(want) & torch.isnan(g) | (g == want) | ((g - want).abs() <= 2.0 ** -23 * want.abs() + E.squeeze(-1) + 2.0 ** -18)
                assert ok.all(), (i, h)
    assert (out[s.total:] == 9.0).all() and (L is None or (L[s.total:] == 9.0).all())
    return q, out, work


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D,H,G,page", [(64, 1, 1, 16), (64, 8, 4, 64), (128, 2, 8, 32), (128, 1, 5, 128), (256, 4, 6, 16), (256, 2, 1, 64), (128, 1, 17, 16)])
def test_attention_one_token(gpu, lb, D, H, G, page, t):
    s = Setup(lb, [(1, 0), (1, 1), (1, 15), (0, 9), (1, 16), (1, 63), (1, 64), (1, 500), (1, 1023), (1, 3001)], D, H, page, seed=D + G, padded=1)
    check_attention(lb, s, t, G, spread=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D,H,G,page,layout", [(64, 2, 3, 16, "slice"), (128, 1, 4, 64, "odd"), (256, 1, 6, 16, "slice"), (128, 2, 1, 32, "apart")])
def test_attention_ragged_rows(gpu, lb, D, H, G, page, layout, t):
    s = Setup(lb, [(2, 0), (5, 3), (33, 0), (1, 200), (0, 0), (64, 64), (129, 31), (7, 1025)], D, H, page, seed=D + G, padded=3)
    check_attention(lb, s, t, G, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,G,page", [(64, 2, 3, 16), (128, 2, 4, 64), (256, 4, 6, 16)])
def test_attention_trees(gpu, lb, D, H, G, page):
    s = Setup(lb, [(20, 300), (32, 0), (1, 77), (9, 1000), (0, 4), (31, 63)], D, H, page, seed=G, tree=True)
    check_attention(lb, s, "bf16", G)


@pytest.mark.gpu
def test_attention_rows_that_see_nothing(gpu, lb):
    s = Setup(lb, [(6, 0), (4, 50), (32, 0)], 128, 2, 16, seed=5, tree=True)
    for r in (0, 3, 5, 7, 10, 41):
        s.masks[r] = 0  # a row of a sequence without context sees nothing at all
    s.masks[4], s.masks[20] = 1 << 31 | 1 << 5, 1 << 31
    s.anc = torch.tensor([x - (1 << 32) if x >> 31 else x for x in s.masks], dtype=torch.int32).cuda()
    s.masks[4] = 1 << 5  # bits at and past the sequence's rows have no position
    _, out, _ = check_attention(lb, s, "bf16", 2)
    assert (out[0] == 0).all() and (out[10] == 0).all() and not (out[7] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_attention_nan_reaches_only_the_rows_that_see_it(gpu, lb, rows):
    """Every position that no row sees reads as NaN; a NaN key and a NaN value inside the rows reach the rows from there on."""
    s = Setup(lb, [(rows, 70), (rows, 3)], 128, 2, 16, seed=6, fill=0xff)
    n = s.total
    k, v = (torch.randn(n, 2, 128, device="cuda", generator=s.gen) for _ in range(2))
    full = [(r + p, 0) for r, p in s.seqs]
    for i, (m, _) in enumerate(full):  # the context and the rows get values, the rest of the pages stays NaN
        x = torch.randn(m, 2, 128, device="cuda", generator=s.gen)
        b = lb.Kv4Batch(torch.tensor([0, m], dtype=torch.int32, device="cuda"), s.slot[i:i + 1].clone(), torch.zeros(1, dtype=torch.int32, device="cuda"), m, m, m)
        s.cache().append(b, x, x.flip(-1).contiguous())
    if rows > 2:
        page, tok = s.where(0, torch.tensor([70 + rows // 2], device="cuda"))
        s.ks[page, 0, tok] = 0x7f
        page, tok = s.where(1, torch.tensor([3 + rows - 1], device="cuda"))
        s.vs[page, 1, tok] = 0x7f
    _, out, _ = check_attention(lb, s, "bf16", 3)
    nan = torch.isnan(out.float()).any(-1)
    assert nan.sum().item() == (3 * (rows - rows // 2) + 3 if rows > 2 else 0)


@pytest.mark.gpu
def test_attention_infinite_and_nan_queries_stay_in_their_row(gpu, lb):
    s = Setup(lb, [(4, 90)], 64, 1, 16, seed=7)
    q = torch.randn(4, 4, 64, device="cuda", generator=s.gen)
    q[1, 2, 5], q[2, 0, 0] = math.nan, math.nan
    check_attention(lb, s, "bf16", 4, q=q)


@pytest.mark.gpu
def test_attention_extreme_scores_and_tensor_scales(gpu, lb):
    s = Setup(lb, [(1, 2000), (40, 100)], 128, 1, 16, seed=8)
    check_attention(lb, s, "bf16", 4, spread=60.0)                              # one key takes it all
    check_attention(lb, s, "bf16", 4, spread=1.0, k_scale=2.0 ** -6, v_scale=2.0 ** 9, scale=3.0)
    check_attention(lb, s, "f16", 4, spread=1.0, k_scale=2.0 ** 5, v_scale=2.0 ** -9, scale=0.01)
    check_attention(lb, s, "bf16", 4, scale=1e-30)                              # a plain mean
    s.vs.fill_(0x7e)                                                            # the largest values
    check_attention(lb, s, "bf16", 4)


@pytest.mark.gpu
def test_attention_long_context_and_bounds_looser_than_the_lengths(gpu, lb):
    s = Setup(lb, [(1, 70000), (1, 5), (2, 33000)], 64, 2, 64, seed=9, extra_slots=3)
    _, a, _ = check_attention(lb, s, "f16", 8)
    s.gen.manual_seed(1)
    b = Setup(lb, [(1, 300), (3, 5)], 128, 1, 16, seed=10)
    b.tables = torch.cat([b.tables, torch.zeros(b.tables.shape[0], 4000, dtype=torch.int32, device="cuda")], 1)
    b.max_context, b.max_rows = 60000, 4
    b.rows = b.total
    check_attention(lb, b, "bf16", 6)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_scales_below_zero_and_none(gpu, lb, rows):
    s = Setup(lb, [(rows, 90), (rows, 0), (rows, 700)], 64, 2, 16, seed=15 + rows)
    check_attention(lb, s, "bf16", 3, scale=-0.2)
    check_attention(lb, s, "bf16", 3, scale=0.0)                                                        # a plain mean of what a row sees
    check_attention(lb, s, "bf16", 3, scale=1e-30, q=torch.full((s.rows, 6, 64), 1e-30, device="cuda"))  # a product below fp32


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 50])
def test_a_cache_past_32_bits(gpu, lb, rows):
    """The pages in use lie behind 4.9 GB of others in each of k and v."""
    s = Setup(lb, [(rows, 300), (rows, 2000 - rows)], 256, 4, 64, seed=16)
    before = 150000
    for name in ("k", "ks", "v", "vs"):
        x = getattr(s, name)
        y = torch.empty((before + x.shape[0], *x.shape[1:]), dtype=torch.uint8, device="cuda")
        y[before:] = x
        setattr(s, name, y)
    s.tables, s.pages = torch.where(s.tables > 0, s.tables + before, 0), s.pages + before
    assert before * 4 * 64 * 128 > 1 << 32
    check_attention(lb, s, "bf16", 2)
    k, v = (torch.randn(s.rows, 4, 256, device="cuda", generator=s.gen) for _ in range(2))
    got_k, got_v, err = torch.empty_like(k), torch.empty_like(v), torch.zeros(1, dtype=torch.int32, device="cuda")
    s.cache().append(s.batch(), k, v, err=err)
    s.cache().read(s.batch(), got_k, got_v, err=err)
    assert err.item() == 0 and torch.equal(got_k.double(), stored64(k.double())) and torch.equal(got_v.double(), stored64(v.double()))


@pytest.mark.gpu
def test_attention_sequences_that_share_rows_stay_in_bounds(gpu, lb):
    """row0 that descends is against the rules: recorded, and nothing beyond the arrays is touched."""
    H, D, G, n = 1, 64, 8, 20
    s = Setup(lb, [(100, 1100)], D, H, 16, seed=17)
    row0 = torch.tensor([0, 100] * n + [0, 100, 200], dtype=torch.int32, device="cuda")
    seqs = len(row0) - 1
    batch = lb.Kv4Batch(row0, s.slot.repeat(seqs), s.pos.repeat(seqs), 200, 100, 1200)
    q = torch.randn(200, H * G, D, device="cuda", generator=s.gen).bfloat16()
    out = torch.full((202, H * G, D), 9.0, dtype=torch.bfloat16, device="cuda")
    need = s.cache().attention_workspace_bytes(batch, H * G)
    work, err = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    s.cache().attention(batch, q, out[1:201], 0.125, work[:need], err=err)
    assert err.item() == BAD_BATCH and (out[0] == 9.0).all() and (out[201] == 9.0).all() and not work[need:].any()


@pytest.mark.gpu
def test_attention_skips_and_records_bad_pages_and_batches(gpu, lb):
    for bad in (0, "past", -5):
        s = Setup(lb, [(1, 100), (2, 40)], 64, 1, 16, seed=11)
        page = s.pages + 1 if bad == "past" else bad
        s.tables[s.slot[0].long(), 2] = page
        check_attention(lb, s, "bf16", 2, err_code=BAD_PAGE, skip=[0])
    s = Setup(lb, [(1, 100), (2, 40)], 64, 1, 16, seed=12)
    s.slot[0] = -1
    check_attention(lb, s, "bf16", 2, err_code=BAD_BATCH, skip=[0])
    s = Setup(lb, [(1, 100), (2, 40)], 64, 1, 16, seed=12)
    s.max_context = 60  # below the first sequence's 101
    check_attention(lb, s, "bf16", 2, err_code=BAD_BATCH, skip=[0])


@pytest.mark.gpu
def test_attention_workspace_is_left_reusable(gpu, lb):
    """One workspace through calls of other lengths and batches, each as with a fresh one; calls repeat bit for bit."""
    big = Setup(lb, [(1, 9000), (1, 100), (16, 2500)], 128, 2, 16, seed=13)
    cache = big.cache()
    work = torch.zeros(cache.attention_workspace_bytes(big.batch(), 16), dtype=torch.uint8, device="cuda")
    q, out, _ = check_attention(lb, big, "bf16", 8, work=work)
    for seqs in ([(1, 5000)], [(16, 2000), (1, 1)], [(1, 9000), (1, 100), (16, 2500)]):
        s = Setup(lb, seqs, 128, 2, 16, seed=14)
        if s.cache().attention_workspace_bytes(s.batch(), 16) <= work.numel():
            check_attention(lb, s, "bf16", 8, work=work)
    again = torch.zeros_like(out)
    cache.attention(big.batch(), q, again, 1 / math.sqrt(128), work)
    assert torch.equal(again[:big.total], out[:big.total])


# ------------------------------------------------------------------------------------------------ together, streams and graphs
class Layer:
    """One attention layer's decode step in 4 bits: q | k | v projection, append, attention, output projection."""

    def __init__(self, lb, seqs, D=128, H=2, G=4, hidden=512, seed=0, stream=0):
        self.s = Setup(lb, seqs, D, H, 16, seed=seed)
        s, self.lb, self.G, self.D, self.H = self.s, lb, G, D, H
        self.wqkv, self.wo = random_nvfp4(((G + 2) * H * D, hidden), s.gen, 2.0), random_nvfp4((hidden, G * H * D), s.gen, 2.0)
        self.x = torch.randn(s.rows, hidden, device="cuda", generator=s.gen).bfloat16()
        self.qkv = torch.zeros(s.rows, (G + 2) * H * D, dtype=torch.bfloat16, device="cuda")
        self.o, self.y = torch.zeros(s.rows, G * H, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(s.rows, hidden, device="cuda")
        self.cache, self.batch = s.cache(), s.batch()
        self.work = torch.zeros(self.cache.attention_workspace_bytes(self.batch, G * H), dtype=torch.uint8, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(self, stream=0):
        lb, GH, H = self.lb, self.G * self.H, self.H
        lb.nvfp4_matvec(self.x, *self.wqkv, 0.02, self.qkv, stream=stream)
        r = self.qkv.unflatten(1, (-1, self.D))
        q, k, v = r[:, :GH], r[:, GH:GH + H], r[:, GH + H:]
        self.cache.append(self.batch, k, v, q=q, q_out=q, rotary_dim=64, err=self.err, stream=stream)
        self.cache.attention(self.batch, q, self.o, 1 / math.sqrt(self.D), self.work, err=self.err, stream=stream)
        lb.nvfp4_matvec(self.o.flatten(1), *self.wo, 0.02, self.y, stream=stream)

    def want(self):
        s, GH, H, D = self.s, self.G * self.H, self.H, self.D
        qkv = (self.x.double() @ values64(*self.wqkv).t() * 0.02).bfloat16().unflatten(1, (-1, D))
        q = rotated64(qkv[:, :GH], s.at, 64, 1e7).bfloat16().double()
        k, v = stored64(rotated64(qkv[:, GH:GH + H], s.at, 64, 1e7)), stored64(qkv[:, GH + H:].double())
        o = torch.zeros(s.rows, GH, D, device="cuda", dtype=torch.float64)
        for i, (n, p) in enumerate(s.seqs):
            a = int(s.row0[i])
            K, V = s.held(i, n + p)
            K[p:], V[p:] = k[a:a + n], v[a:a + n]
            for h in range(GH):
                sc = (q[a:a + n, h] @ K[:, h // self.G].t() / math.sqrt(D)).masked_fill(~s.visible(i), -math.inf)
                o[a:a + n, h] = torch.softmax(sc, -1) @ V[:, h // self.G]
        return o.bfloat16().double().flatten(1) @ values64(*self.wo).t() * 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 0)], [(1, 33), (1, 700), (1, 5000)], [(5, 16), (20, 333)]])
def test_a_decode_layer(gpu, lb, seqs):
    """All operators in a row.  A rounding of the projection that falls the other way (BF16, 2^-8) can move a code of the cache by a
    step, so the result is held in norm: BF16 roundings of x, q, o (2^-8 each, independent) and codes that differ."""
    L = Layer(lb, seqs)
    L.step()
    assert L.err.item() == 0
    want = L.want()
    assert ((L.y.double() - want).norm() / want.norm()).item() < 4 * 2.0 ** -8


@pytest.mark.gpu
def test_on_another_stream_and_captured(gpu, lb):
    L = Layer(lb, [(1, 40), (1, 900)])
    L.step()
    torch.cuda.synchronize()
    want = L.y.clone()
    side = torch.cuda.Stream()
    L.y.zero_()
    side.wait_stream(torch.cuda.current_stream())
    L.step(side.cuda_stream)
    side.synchronize()
    assert torch.equal(L.y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.step(torch.cuda.current_stream().cuda_stream)
    L.y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(L.y, want)
    # the graph reads the batch when it runs: the next tokens, one position on
    L.s.pos += 1
    L.s.seqs = [(1, 41), (1, 901)]
    L.s.at = L.s.at + 1
    L.x.normal_()
    g.replay()
    torch.cuda.synchronize()
    assert L.err.item() == BAD_BATCH  # beyond the host's bound on the context: refused on the device, recorded
    L.err.zero_()


@pytest.mark.gpu
def test_two_graphs_at_once_with_a_workspace_each(gpu, lb):
    a, b = Layer(lb, [(1, 6000), (3, 50)], seed=1), Layer(lb, [(1, 4000), (2, 800)], seed=2)
    wants, graphs = [], []
    for L in (a, b):
        L.step()
        torch.cuda.synchronize()
        wants.append(L.y.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            L.step(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.y, wants[0]) and torch.equal(b.y, wants[1])
