"""Calls at the limits of the operators of a decode layer in 4 bits: sizes at which an index would leave 32 bits, batches against the
rules, contexts so long that a sum's roundings add up, values on a rounding's border.  Refusals are checked without a GPU."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from test_decode4 import BAD_BATCH, Setup, T, c_batch, c_cache, calls, check_attention, e4m3_table, matvec_case, random_nvfp4, rotated64, stored64, values64, _p  # noqa: E402


# ------------------------------------------------------------------------------------------------ refusals, without a GPU
def matvec_status(lb, M, N, K, xt):
    fn = lb.lib().ling_b200_nvfp4_matvec
    fn.argtypes = lb._MATVEC_ARGS
    return fn(0, _p(), xt, K, M, _p(2), _p(3), 1.0, N, K, _p(4), lb.F32, N, 0, None)


@pytest.mark.parametrize("K", [57344 + 16, 1 << 20, 1 << 25, 34000000, (1 << 31) - 16])
def test_matvec_refuses_activations_beyond_shared_memory(lb, K):
    """Before any plan is made: at K = 2^25 the activations of 32 columns are 2^31 bytes."""
    for M, xt in ((8, lb.BF16), (32, lb.BF16), (32, lb.F16), (4, lb.F32), (32, lb.F32)):
        assert matvec_status(lb, M, 8, K, xt) == lb.ERR_UNSUPPORTED and "shared memory" in lb.last_error()
    if K > 462848:
        assert matvec_status(lb, 1, 8, K, lb.BF16) == lb.ERR_UNSUPPORTED


def test_matvec_refuses_rows_of_weights_beyond_32_bits(lb):
    for N in ((1 << 31) - 1, (1 << 31) - 31):
        assert matvec_status(lb, 1, N, 16, lb.BF16) == lb.ERR_ARG and lb.last_error()


@pytest.mark.parametrize("rows,G", [(1 << 24, 128), (1 << 22, 512), (1 << 21, 1024), ((1 << 24) - 1, 1024)])
def test_attention_refuses_query_rows_beyond_32_bits(lb, rows, G):
    """rows x heads of a group: counted in 32 bits by the kernels (an output of this size is beyond any device)."""
    cache, batch = c_cache(lb, kv_heads=1, max_pages=1 << 20), c_batch(lb, rows=rows, max_rows=rows, max_context=rows)
    out = (8192, G * 128, 128)
    assert calls(lb, cache, batch, q_heads=G, q=(4096, G * 128, 128), out=out, ws=1 << 62)[2] == lb.ERR_ARG and "q_heads / kv_heads" in lb.last_error()
    assert lb.lib().ling_b200_kv4_attention_workspace(C.byref(cache), C.byref(batch), G) == 0


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.gpu
@pytest.mark.parametrize("M,K,xt", [(8, 57344, "bf16"), (32, 57344, "f16"), (5, 57328, "f32"), (1, 462848, "bf16"), (2, 230016, "f16")])
def test_matvec_longest_reductions(gpu, lb, M, K, xt):
    """The longest K that a row count takes, and launches of eight columns each where there are more."""
    matvec_case(lb, M, 100, K, xt, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,xt", [(16, 34979, 5120, "f16"), (32, 34979, 5120, "bf16"), (16, 34979, 5120, "f32"), (1, 30011, 8208, "bf16"), (8, 70001, 2064, "f32"),
                                      (4, 34979, 12304, "f32"), (20, 5123, 17408, "bf16"), (3, 20011, 17408, "f16"), (32, 1003, 17408, "f16"), (29, 517, 17408, "f32"),
                                      (9, 5003, 12304, "f32")])
def test_matvec_many_meetings_and_launches(gpu, lb, M, N, K, xt):
    """More tiles than sums have room for, so that CTAs (and a CTA's warps) meet several times, with a rest; rows that take several launches.
    Calls repeat bit for bit."""
    x, w, ws, y = matvec_case(lb, M, N, K, xt, "f32")
    for _ in range(5):
        again = torch.zeros_like(y)
        lb.nvfp4_matvec(x, w, ws, 0.37, again)
        assert torch.equal(again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(1, 16), (5, 16), (40, 16), (33, 48), (17, 272), (75, 1088), (64, 5120), (37, 3344)])
def test_matvec_scales_from_any_byte_on(gpu, lb, N, K):
    """Scales inside a larger array, from every kind of byte on: as the same scales on a boundary, whatever lies around them."""
    gen = torch.Generator("cuda").manual_seed(N + K)
    w, ws = random_nvfp4((N, K), gen)
    for M in (1, 9):
        x = torch.randn(M, K, device="cuda", generator=gen).bfloat16()
        want = torch.zeros(M, N, device="cuda")
        lb.nvfp4_matvec(x, w, ws, 0.5, want)
        assert torch.isfinite(want).all()
        for off in (1, 2, 7, 15, 16):
            around = torch.full((off + ws.numel() + 40,), 0x7f, dtype=torch.uint8, device="cuda")  # NaN
            inside = around[off:off + ws.numel()].view(N, K // 16)
            inside.copy_(ws)
            got = torch.zeros(M, N, device="cuda")
            lb.nvfp4_matvec(x, w, inside, 0.5, got)
            assert torch.equal(got, want), (M, off)


@pytest.mark.gpu
@pytest.mark.parametrize("xt", ["bf16", "f32", "f16"])
def test_matvec_elements_far_below_their_rows_largest(gpu, lb, xt):
    """The largest elements meet weights of 0: what is left of the others is off by 2^-39 of the largest each (FP16: by nothing)."""
    gen = torch.Generator("cuda").manual_seed(3)
    w, ws = random_nvfp4((64, 512), gen)
    w[:, ::16] = 0  # codes of k = 0, 1, 32, 33, ..
    for far in (0, 10, 20, 30):
        x = torch.randn(4, 512, device="cuda", generator=gen)
        x.unflatten(1, (-1, 32))[:, :, :2] *= 2.0 ** (min(far, 14) if xt == "f16" else far)
        x = x.to(T[xt])
        y = torch.zeros(4, 64, device="cuda")
        lb.nvfp4_matvec(x, w, ws, 1.0, y)
        x64, w64 = x.double(), values64(w, ws)
        tol = 2.0 ** -23 * (512 / 16 + 64) * (x64.abs() @ w64.abs().t()) + (xt != "f16") * 2.0 ** -39 * x64.abs().amax(1, keepdim=True) * w64.abs().sum(1)
        assert ((y.double() - x64 @ w64.t()).abs() <= tol).all(), far


# ------------------------------------------------------------------------------------------------ batches against the rules
DESCENDING = [[0, 9, 2, 3], [0, 10, 2, 3, 12], [0, 2, 12, 11], [3, 0, 12], [0] + [2] * 60 + [12, 5, 12]]


@pytest.mark.gpu
@pytest.mark.parametrize("row0", DESCENDING)
def test_append_and_read_skip_a_batch_whose_row0_descends(gpu, lb, row0):
    """Its rows lie in several sequences, or would be counted to one that does not hold them, positions behind its own rows."""
    s = Setup(lb, [(12, 50)], 64, 2, 16, fill=0x11, padded=2)
    n = len(row0) - 1
    batch = lb.Kv4Batch(torch.tensor(row0, dtype=torch.int32, device="cuda"), s.slot.repeat(n), s.pos.repeat(n), s.rows, 12, s.max_context)
    x = torch.randn(s.rows, 2, 64, device="cuda", generator=s.gen)
    out, err = torch.full_like(x, 9.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    s.cache().append(batch, x, x, q=x, q_out=out, rotary_dim=64, err=err)
    assert err.item() == BAD_BATCH and (out == 9.0).all() and all((a == 0x11).all() for a in (s.k, s.ks, s.v, s.vs))
    err.zero_()
    s.cache().read(batch, out, None, err=err)
    assert err.item() == BAD_BATCH and (out == 9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["behind the rows", "slot of none", "position of none"])
def test_append_and_read_record_sequences_that_no_row_meets(gpu, lb, what):
    """As the attention does: a sequence that starts behind the arrays' rows, or has no rows, and is outside the bounds."""
    s = Setup(lb, [(5, 20), (3, 40)], 64, 1, 16, fill=0x11) if what == "behind the rows" else Setup(lb, [(5, 20), (0, 40)], 64, 1, 16, fill=0x11)
    s.rows = 5
    if what == "slot of none":
        s.slot[1] = -1
    elif what == "position of none":
        s.pos[1] = s.max_context + 1
    x = torch.randn(5, 1, 64, device="cuda", generator=s.gen)
    out, q, err = torch.full_like(x, 9.0), torch.zeros(5, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    s.cache().append(s.batch(), x, x, err=err)
    assert err.item() == BAD_BATCH
    err.zero_()
    s.cache().read(s.batch(), out, None, err=err)
    assert err.item() == BAD_BATCH and torch.equal(out.double(), stored64(x.double()))
    err.zero_()
    work = torch.zeros(s.cache().attention_workspace_bytes(s.batch(), 2), dtype=torch.uint8, device="cuda")
    s.cache().attention(s.batch(), q, torch.zeros_like(q), 0.1, work, err=err)
    assert err.item() == BAD_BATCH


@pytest.mark.gpu
def test_rows_beyond_a_bound_of_none_are_recorded(gpu, lb):
    """max_rows = 0 and a sequence with rows: outside the bounds, by every call; without rows there is nothing to record."""
    for seqs, want in (([(3, 20), (0, 5)], BAD_BATCH), ([(0, 20), (0, 5)], 0)):
        s = Setup(lb, seqs, 64, 1, 16, padded=5 - sum(r for r, _ in seqs))
        s.max_rows = 0
        x, q = torch.randn(5, 1, 64, device="cuda", generator=s.gen), torch.zeros(5, 2, 64, dtype=torch.bfloat16, device="cuda")
        out, o, err = torch.full_like(x, 9.0), torch.full_like(q, 9.0), torch.zeros(3, dtype=torch.int32, device="cuda")
        s.cache().append(s.batch(), x, x, err=err[:1])
        s.cache().read(s.batch(), out, None, err=err[1:2])
        work = torch.zeros(s.cache().attention_workspace_bytes(s.batch(), 2), dtype=torch.uint8, device="cuda")
        s.cache().attention(s.batch(), q, o, 0.1, work, err=err[2:])
        assert err.tolist() == [want] * 3 and (out == 9.0).all() and (o == 9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("G", [2, 8, 40])
@pytest.mark.parametrize("row0", DESCENDING)
def test_attention_skips_a_batch_whose_row0_descends(gpu, lb, row0, G):
    """By either kernel, with split contexts and without."""
    for pos, far in ((50, 0), (50, 1500), (3000, 0)):
        s = Setup(lb, [(12, pos)], 64, 1, 16, fill=0x11, padded=2, slack=0)
        n = len(row0) - 1
        if far:  # (a bound on the context that lets the host split it)
            s.tables, s.max_context = torch.cat([s.tables, s.tables[:, :1].repeat(1, 100)], 1), far
        batch = lb.Kv4Batch(torch.tensor(row0, dtype=torch.int32, device="cuda"), s.slot.repeat(n), s.pos.repeat(n), s.rows, 12, s.max_context)
        q = torch.randn(s.rows, G, 64, device="cuda", generator=s.gen).bfloat16()
        out, lse, err = torch.full_like(q, 9.0), torch.full((s.rows, G), 9.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        work = torch.full((s.cache().attention_workspace_bytes(batch, G),), 0x3f, dtype=torch.uint8, device="cuda")
        s.cache().attention(batch, q, out, 0.125, work, lse=lse, err=err)
        assert err.item() == BAD_BATCH and (out == 9.0).all() and (lse == 9.0).all()


# ------------------------------------------------------------------------------------------------ roundings
@pytest.mark.gpu
@pytest.mark.parametrize("rows,G", [(1, 4), (40, 2)])
def test_attention_nan_beside_scores_that_underflow(gpu, lb, rows, G):
    """A row sees a NaN key (or value) whose split counts for nothing beside another split's score: NaN times 0 is NaN."""
    for which in ("k", "v"):
        s = Setup(lb, [(rows, 3000), (rows, 2900)], 128, 1, 16, seed=21)
        page, tok = s.where(0, torch.tensor([2990], device="cuda"))
        key = s.held(0, 3000)[0][2990]  # [H][D]
        q = torch.cat([12.0 * key.float().expand(rows, G, 128), torch.randn(rows, G, 128, device="cuda", generator=s.gen)])
        page, tok = s.where(0, torch.tensor([5], device="cuda"))
        (s.ks if which == "k" else s.vs)[page, 0, tok] = 0x7f
        _, out, _ = check_attention(lb, s, "bf16", G, q=q)
        assert torch.isnan(out[:rows]).all() and torch.isfinite(out[rows:2 * rows]).all()


def constant_values(lb, kind, D, n):
    """Attention over n positions whose V is one vector: (output, that vector).  Each probability is off by half an FP16 step at most."""
    seqs, rows, G = {"warps alone": (1024, 1, 16), "warps together": (73, 1, 4), "tiles": (1, 1200, 16)}[kind]
    page, gen = 64, torch.Generator("cuda").manual_seed(n + D)
    pages = -(-(n + rows) // page)
    k = torch.randint(0, 256, (pages + 1, 1, page, D // 2), dtype=torch.uint8, device="cuda", generator=gen)
    ks = torch.full((pages + 1, 1, page, D // 16), 0x30, dtype=torch.uint8, device="cuda")  # 1/2
    v_one = torch.randint(0, 256, (D // 2,), dtype=torch.uint8, device="cuda", generator=gen)
    vs_one = (0x38 + torch.arange(D // 16, device="cuda") % 8).to(torch.uint8)
    v, vs = v_one.expand(pages + 1, 1, page, D // 2).contiguous(), vs_one.expand(pages + 1, 1, page, D // 16).contiguous()
    tables = torch.arange(1, pages + 1, dtype=torch.int32, device="cuda").view(1, -1)
    cache = lb.Kv4Cache(k, ks, v, vs, tables)
    full = lambda x: torch.full((seqs,), x, dtype=torch.int32, device="cuda")
    batch = lb.Kv4Batch(torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * rows, full(0), full(n), seqs * rows, rows, n + rows)
    q = torch.randn(seqs * rows, G, D, device="cuda", generator=gen).half()
    out, err = torch.zeros_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    work = torch.empty(cache.attention_workspace_bytes(batch, G), dtype=torch.uint8, device="cuda")
    cache.attention(batch, q, out, 1 / math.sqrt(D), work, err=err)
    assert err.item() == 0
    return out.double(), values64(v_one, vs_one)


def check_constant_values(lb, kind, D, n):
    """out = V.  Half an FP16 step each for the output and the probabilities, and what a chain of tensor-core sums loses: at most 2^-23 of
    the sum a link of 16 positions, which must not go on over the whole context (at n = 2^20 that would be up to 2^-7): 2^-14 for 512 links."""
    out, v = constant_values(lb, kind, D, n)
    off = ((out - v).abs() / v.abs().clamp(min=2.0 ** -10)).max().item()
    assert off <= 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -14, off


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["warps alone", "warps together"])
@pytest.mark.parametrize("D,n", [(64, 1 << 20), (128, 300001), (256, 1 << 19), (256, 4097), (64, 4095)])
def test_attention_sums_over_long_contexts_of_a_warp(gpu, lb, kind, D, n):
    check_constant_values(lb, kind, D, n)


@pytest.mark.gpu
@pytest.mark.parametrize("D,n", [(64, 1 << 20), (128, 300001), (256, 1 << 19), (256, 8193), (64, 8192 - 1200)])
def test_attention_sums_over_long_contexts_of_a_tile(gpu, lb, D, n):
    check_constant_values(lb, "tiles", D, n)


@pytest.mark.gpu
def test_append_scales_beside_a_rounding_border(gpu, lb):
    """Rotated keys whose largest value over 6 lies 2^-27 of itself beside the middle of two E4M3 values: the scale is the exact quotient's,
    not that of its fp32 rounding, which is the middle itself."""
    tab = e4m3_table()[:127]
    lows = torch.tensor([c for c in range(0x30, 0x50)])
    middle = (tab[lows] + tab[lows + 1]) / 2
    want = torch.cat([middle * 6 * (1 + d) for d in (2.0 ** -27, -2.0 ** -27)])  # the group's largest value
    n, D, p = len(want), 64, 1
    c, sn = math.cos(p), math.sin(p)
    x = (want / c).float()  # dims 0 and 32 turn together by p: x cos p - o sin p, o making up for what fp32 rounded off x
    o = ((x.double() * c - want) / sn).float()
    k = torch.full((n, 1, D), 0.125)
    k[:, 0, 0], k[:, 0, 32] = x, o
    turned = rotated64(k, torch.full((n,), p), D, 1e7)
    top = turned[:, 0, :16].abs().amax(-1)
    assert (turned[:, 0, 0].abs() == top).all() and ((top / want - 1).abs() < 2.0 ** -40).all() and torch.equal((top / 6).float().double(), torch.cat([middle, middle]))
    k = k.cuda()
    s = Setup(lb, [(1, p)] * n, D, 1, 16, fill=0)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s.cache().append(s.batch(), k, k, rotary_dim=D, theta=1e7, err=err)
    page, tok = s.tables[s.slot.long(), 0].long(), p
    got = s.ks[page, 0, tok, 0].cpu().long()
    assert err.item() == 0 and torch.equal(got, torch.cat([lows + 1, lows]))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,G", [([(600, 20000), (600, 17000)], 8), ([(1, 50000 - 100 * i) for i in range(100)], 24)])
def test_attention_scores_that_grow_from_chain_to_chain(gpu, lb, seqs, G):
    """Keys whose size grows along the context, so that the reference moves after a chain has ended; a NaN value in the last sequence's
    first chain."""
    s = Setup(lb, seqs, 64, 1, 64, seed=23)
    for i, (r, p) in enumerate(seqs):
        n = -(-(r + p) // 64)
        s.ks[s.tables[s.slot[i].long(), :n].long()] = (0x10 + 40 * torch.arange(n, device="cuda") // n).to(torch.uint8)[:, None, None, None]
    page, tok = s.where(len(seqs) - 1, torch.tensor([5], device="cuda"))
    s.vs[page, 0, tok] = 0x7f
    _, out, _ = check_attention(lb, s, "bf16", G, spread=2.0, lse=False)
    last = seqs[-1][0]
    assert torch.isnan(out[-last:]).all() and torch.isfinite(out[:-last]).all()


# ------------------------------------------------------------------------------------------------ lopsided batches
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 256])
def test_attention_one_long_context_among_empty_sequences(gpu, lb, D):
    """Bounds that speak for many items, and one item: its context is shared by hundreds of warps."""
    s = Setup(lb, [(0, 3)] * 50 + [(1, 120000)] + [(0, 0)] * 49, D, 1, 64, seed=31, padded=1)
    check_attention(lb, s, "bf16", 3, spread=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("bad", [0, 20, 39, 69])
def test_attention_records_a_bad_sequence_among_many(gpu, lb, bad, G):
    """Wherever it stands, by either kernel; the others get their results."""
    s = Setup(lb, [(1 + i % 7, 40 + 13 * i) for i in range(70)], 64, 1, 16, seed=32)
    s.slot[bad] = s.tables.shape[0]
    check_attention(lb, s, "bf16", G, err_code=BAD_BATCH, skip=[bad])
