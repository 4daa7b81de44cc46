"""Batched serving operators (polarflash_b200.serving): the paged cache write,
attention over pages, attention of packed prompts and the draw of a token,
each against its definition in 64 bits.

Tolerances, from the roundings on the way:
- cache write: rotation and quantization are separate fp32 operations in a
  fixed order, so outputs and codes are equal bit for bit;
- attention of one token (fp32 sums): a score is off by a few 2^-22 of
  sum |q k| scale, below 32 here, so weights are off by < 32 * 2^-21 = 1.6e-5
  relative, and so is the output against sum p |v|; rounding to 16 bits
  adds half a step of the output (bf16 2^-8, fp16 2^-11 of |out|);
- prompt attention: each weight is rounded once to 16 bits before it meets v
  (half a step e of p |v|), the weight from an exponential good to 2^-10 of
  that step's type or better, and the output once (e |out| <= e sum p |v|):
  2 e + e / 2 + 1.6e-5 of sum p |v|, e = 2^-8 (bf16) or 2^-11 (fp16), plus the
  smallest fp16 step 2^-24 where weights underflow, times the key count;
- the drawn token: equal."""
import ctypes
import math

import pytest
import torch

from polarflash_b200 import _lib

gpu = pytest.mark.gpu
MODES = ("fp16", "bf16", "int8", "2bit", "2bit_asym")
HALF_STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
A = 0x100000  # an aligned stand-in address


def _api():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import polarflash_b200 as P

    return P


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- on the host ---------------------------------------------------------------
def _pages_desc(**kw):
    f = dict(mode=1, num_pages=4, page_size=16, n_kv_heads=2, head_dim=64, k=A, v=A, k_scales=A, v_scales=A, k_zeros=None,
             v_zeros=None)
    f.update(kw)
    d = _lib.PFKVPages()
    for k, v in f.items():
        setattr(d, k, v)
    return d


def test_page_descriptor_is_checked_on_the_host():
    c = lambda **kw: _lib.load().pf_kv_pages_check(ctypes.byref(_pages_desc(**kw)))  # noqa: E731
    assert c() == _lib.OK
    assert _lib.load().pf_kv_pages_check(None) == _lib.ERR_INVALID_ARGUMENT
    for bad in (dict(mode=0), dict(mode=4), dict(k=None), dict(v=None), dict(k_scales=None), dict(mode=3),
                dict(mode=3, k_zeros=A)):
        assert c(**bad) == _lib.ERR_INVALID_ARGUMENT, bad
    assert c(mode=3, k_zeros=A, v_zeros=A) == _lib.OK
    assert c(mode=8, k_scales=None, v_scales=None) == _lib.OK
    for bad in (dict(num_pages=0), dict(n_kv_heads=0), dict(head_dim=96), dict(page_size=8), dict(page_size=48),
                dict(page_size=512)):
        assert c(**bad) == _lib.ERR_SHAPE, bad
    for bad in (dict(k=A + 8), dict(v=A + 2), dict(k_scales=A + 4), dict(mode=3, k_zeros=A + 4, v_zeros=A)):
        assert c(**bad) == _lib.ERR_ALIGNMENT, bad


def test_serving_entry_points_refuse_on_the_host():
    L = _lib.load()
    launches = L.pf_kernel_launches()
    I, S, AL, W = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_SHAPE, _lib.ERR_ALIGNMENT, _lib.ERR_WORKSPACE
    pg = ctypes.byref(_pages_desc())

    def rope(pages=pg, q=A, qs=256, k=A, ks=128, v=A, vs=128, dt=0, cos=A, sin=A, T=3, cu=A, lens=A, table=A, width=2,
             seqs=2, nh=4, qo=A, ko=None, vo=None, odt=0):
        return L.pf_paged_rope_kv(pages, q, qs, k, ks, v, vs, dt, cos, sin, T, cu, lens, table, width, seqs, nh, qo, ko,
                                  vo, odt, None)

    assert rope(T=0) == _lib.OK and rope(seqs=0) == _lib.OK  # nothing to do
    for bad in (dict(k=None), dict(lens=None), dict(table=None), dict(sin=None), dict(q=None), dict(qo=None), dict(nh=0),
                dict(ko=A), dict(dt=3), dict(odt=7), dict(T=-1), dict(seqs=-1), dict(odt=1), dict(qs=512)):
        assert rope(**bad) == I, bad  # the last two: q itself as output, of another type or strided
    for bad in (dict(width=0), dict(cu=None), dict(qs=252), dict(ks=124), dict(vs=64), dict(T=0x7fffffff)):
        assert rope(**bad) == S, bad
    for bad in (dict(qo=A + 8), dict(k=A + 4), dict(cos=A + 4), dict(lens=A + 2), dict(ks=130), dict(cu=A + 1)):
        assert rope(**bad) == AL, bad
    need = L.pf_paged_attention_workspace_size(4, 2, 64, 2)
    assert need > 0 and L.pf_paged_attention_workspace_size(3, 2, 64, 2) == 0

    def att(pages=pg, q=A, dt=0, out=A, table=A, width=2, lens=A, seqs=2, nh=4, scale=0.1, ws=A, wsb=need):
        return L.pf_paged_attention(pages, q, dt, out, table, width, lens, seqs, nh, scale, ws, wsb, None)

    assert att(seqs=0) == _lib.OK
    for bad in (dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(ws=None), dict(dt=5), dict(seqs=-1),
                dict(scale=math.nan)):
        assert att(**bad) == I, bad
    for bad in (dict(nh=3), dict(nh=0), dict(width=0), dict(seqs=0x7fffffff)):
        assert att(**bad) == S, bad
    assert att(q=A + 8) == AL and att(ws=A + 8) == AL and att(wsb=need - 1) == W
    assert att(pages=ctypes.byref(_pages_desc(head_dim=80))) == S

    def prompt(q=A, qs=256, k=A, ks=128, v=A, vs=128, out=2 * A, os=256, dt=1, cq=A, ck=A, seqs=2, tq=5, tk=5, nh=4, nkv=2,
               hd=64, scale=0.1):
        return L.pf_prompt_attention(q, qs, k, ks, v, vs, out, os, dt, cq, ck, seqs, tq, tk, nh, nkv, hd, scale, None, None)

    assert prompt(seqs=0) == _lib.OK and prompt(tq=0) == _lib.OK
    for bad in (dict(q=None), dict(k=None), dict(out=None), dict(out=A), dict(cq=None), dict(ck=None), dict(dt=0), dict(tq=-1),
                dict(scale=math.nan), dict(scale=0.0), dict(scale=math.inf)):
        assert prompt(**bad) == I, bad
    for bad in (dict(nh=3), dict(hd=68), dict(hd=136, qs=1024, ks=512, vs=512, os=1024), dict(qs=248), dict(ks=120),
                dict(os=128), dict(nkv=0)):
        assert prompt(**bad) == S, bad
    for bad in (dict(q=A + 8), dict(out=A + 2), dict(qs=260), dict(vs=130), dict(cq=A + 2)):
        assert prompt(**bad) == AL, bad

    def draw(l=A, stride=100, dt=0, rows=2, vocab=100, u=A, ts=None, out=A):
        return L.pf_sample_logits(l, stride, dt, rows, vocab, u, ts, 1.0, None, 0, None, 1.0, None, 0.0, out, None)

    assert draw(rows=0) == _lib.OK
    for bad in (dict(l=None), dict(u=None), dict(out=None), dict(dt=4), dict(rows=-1)):
        assert draw(**bad) == I, bad
    for bad in (dict(vocab=0), dict(vocab=360001, stride=360001), dict(stride=99)):
        assert draw(**bad) == S, bad
    for bad in (dict(l=A + 2), dict(u=A + 1), dict(ts=A + 2), dict(out=A + 4)):
        assert draw(**bad) == AL, bad
    assert L.pf_kernel_launches() == launches


# ---- pages ------------------------------------------------------------------------
def _values(pages, which):
    """The fp64 values of the cache's rows [num_pages, kv_heads, page_size, head_dim]."""
    c = getattr(pages, which)
    if pages.mode in ("fp16", "bf16"):
        return c.double()
    s, z = getattr(pages, which + "_scales").double()[..., None], getattr(pages, which + "_zeros")
    if pages.mode == "int8":
        return c.double() * s
    c = torch.stack([(c >> sh & 3) for sh in (6, 4, 2, 0)], -1).flatten(-2).double()
    return (c - 1.5) * s if pages.mode == "2bit" else c * s + z.double()[..., None]


def _quantize(x, mode):
    """Codes, scales and zeros of rows x [..., hd] (fp32), operation by operation."""
    inv = lambda v: torch.tensor(1.0, device=x.device) / torch.tensor(v, device=x.device)  # noqa: E731
    small = torch.tensor(1e-8, device=x.device)
    z = None
    if mode == "int8":
        s = torch.maximum(x.abs().amax(-1) * inv(127.0), small)
        return torch.round(x / s[..., None]).clamp(-128, 127).to(torch.int8), s, z
    if mode == "2bit":
        s = torch.maximum(x.abs().amax(-1) * inv(1.75), small)
        c = torch.floor(x / s[..., None] + 2.0)
    else:
        z = x.amin(-1)
        s = torch.maximum((x.amax(-1) - z) * inv(3.0), small)
        c = torch.round((x - z[..., None]) / s[..., None])
    c = c.clamp(0, 3).to(torch.uint8).unflatten(-1, (-1, 4))
    return (c[..., 0] << 6) | (c[..., 1] << 4) | (c[..., 2] << 2) | c[..., 3], s, z


def _filled(P, mode, num_pages, page, nkv, hd, g, spread=1.0):
    pg = P.KVPages.empty(mode, num_pages, page, nkv, hd, "cuda")
    for which in ("k", "v"):
        x = torch.randn(num_pages, nkv, page, hd, generator=g, device="cuda")
        x *= torch.exp(spread * torch.randn(num_pages, nkv, page, 1, generator=g, device="cuda"))
        if which == "k":
            x = x.clamp(-6, 6)
        if mode in ("fp16", "bf16"):
            getattr(pg, which).copy_(x)
        else:
            from polarflash_b200.kv_cache import kv_quantize

            c, s, z = kv_quantize(x, mode)
            getattr(pg, which).copy_(c)
            getattr(pg, which + "_scales").copy_(s[..., 0])
            if z is not None:
                getattr(pg, which + "_zeros").copy_(z[..., 0])
    return pg


def _block_table(lens, page, num_pages, g, width=None):
    need = [-(-n // page) for n in lens]
    order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t


def _attend64(pages, q, table, lens, scale):
    """(out, sum p |v|) in fp64, positions of pages outside the cache left out."""
    k, v = _values(pages, "k"), _values(pages, "v")
    out, mag = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    G = q.shape[1] // pages.kv_heads
    for b, n in enumerate(lens):
        pos = torch.arange(max(0, min(n, table.shape[1] * pages.page_size)), device="cuda")
        at = table[b].long()[pos // pages.page_size]
        ok = (at >= 0) & (at < pages.num_pages)
        at, pos = at[ok], pos[ok]
        if len(pos) == 0:
            continue
        kk, vv = (x[at, :, pos % pages.page_size] for x in (k, v))  # [n, nkv, hd]
        for h in range(q.shape[1]):
            p = torch.softmax(kk[:, h // G] @ q[b, h].double() * scale, 0)
            out[b, h], mag[b, h] = p @ vv[:, h // G], p @ vv[:, h // G].abs()
    return out, mag


def _near(got, want, mag, rel):
    off = (got.double() - want).abs()
    bound = rel * mag + HALF_STEP[got.dtype] * want.abs() + 1e-30
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), float((off / bound).max())


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hd,page,dt,odt", [(128, 16, torch.float32, torch.bfloat16), (64, 64, torch.float32, torch.float32),
                                            (128, 32, torch.bfloat16, torch.bfloat16), (64, 16, torch.float16, torch.float32)])
def test_cache_write_is_bit_exact(mode, hd, page, dt, odt):
    """Ragged prompts on cached prefixes, rows behind the last sequence, an
    empty sequence, a position behind the table, pages outside the cache and
    fewer cached tokens than new ones: rows that have a place are equal to the
    fp32 formulas, all others keep their bytes."""
    P = _api()
    g = _gen(hd + page)
    nh, nkv, N = 6, 2, 40
    pages = _filled(P, mode, N, page, nkv, hd, g)
    new, past = [5, 0, 1, page + 3, 7, 2], [0, 9, page - 1, 2 * page - 2, 0, 0]
    lens = [a + b for a, b in zip(new, past)]
    table = _block_table(lens, page, N - 4, g, width=4)
    table[4, 0] = N  # not a page
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lens_t[5] = 1  # two new tokens, one place: the first has position -1
    cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    T = sum(new) + 3  # three rows behind the last sequence
    wide = torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(dt)
    q, k, v = (t.unflatten(1, (-1, hd)) for t in wide.split([nh * hd, nkv * hd, nkv * hd], 1))
    ang = torch.rand(T, hd // 2, generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    names = [n for n in ("k", "v", "k_scales", "v_scales", "k_zeros", "v_zeros") if getattr(pages, n) is not None]
    want = {n: getattr(pages, n).clone() for n in names}
    qo, ko, vo = P.paged_rope_kv(q, k, v, cos, sin, pages, table, lens_t, cu, out_dtype=odt, return_kv=True)

    def turn(x):
        x = x.float()
        a, b, c, s = x[..., : hd // 2], x[..., hd // 2:], cos[:, None], sin[:, None]
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    n = sum(new)
    kr, vr = turn(k), v.float()
    for got, ref in ((qo, turn(q)), (ko, kr), (vo, vr)):
        assert torch.equal(got[:n], ref[:n].to(odt))
    t = 0
    for b, m in enumerate(new):
        for j in range(m):
            pos, t = int(lens_t[b]) - m + j, t + 1
            if pos < 0 or pos // page >= 4 or not 0 <= int(table[b, pos // page]) < N:
                continue
            at = (int(table[b, pos // page]), slice(None), pos % page)
            for which, x in (("k", kr[t - 1]), ("v", vr[t - 1])):
                if mode in ("fp16", "bf16"):
                    want[which][at] = x.to(want[which].dtype)
                    continue
                c, s, z = _quantize(x, mode)
                want[which][at], want[which + "_scales"][at] = c, s
                if z is not None:
                    want[which + "_zeros"][at] = z
    for name in names:
        assert torch.equal(getattr(pages, name), want[name]), name


@gpu
@pytest.mark.parametrize("mode", ["int8", "2bit", "2bit_asym"])
def test_cache_write_at_borders(mode):
    """Values on and next to the borders between codes, tiny and huge rows, zeros:
    codes are those of the rounded quotient."""
    P = _api()
    g = _gen(6)
    T, nkv, hd = 4096, 2, 128
    step = {"int8": 1 / 254, "2bit": 1 / 3.5, "2bit_asym": 1 / 6}[mode]  # halves of a step, of the largest
    k = torch.randint(-300, 300, (T, nkv, hd), generator=g, device="cuda").float() * step
    k[:, :, 0], k[:, :, 1] = (1.0, -1.0) if mode != "2bit_asym" else (1.0, 0.0)
    k = k.clamp(-1 if mode != "2bit_asym" else 0, 1)
    ulp = torch.randint(-2, 3, k.shape, generator=g, device="cuda", dtype=torch.int32)
    k = (k.view(torch.int32) + ulp * (k != 0)).view(torch.float32)
    k = k * torch.exp2(torch.randint(-40, 60, (T, nkv, 1), generator=g, device="cuda").float()) * (
        1 + torch.rand(T, nkv, 1, generator=g, device="cuda"))
    k[0], k[1] = 0.0, 1e-30
    v = k.flip(0).contiguous()
    pages = P.KVPages.empty(mode, T // 64, 64, nkv, hd, "cuda")
    table = torch.arange(T // 64, dtype=torch.int32, device="cuda")[None]
    P.paged_rope_kv(None, k, v, None, None, pages, table, torch.tensor([T], dtype=torch.int32, device="cuda"), _cu([T]))
    for which, x in (("k", k), ("v", v)):
        c, s, z = _quantize(x, mode)
        for name, want in ((which, c), (which + "_scales", s), (which + "_zeros", z)):
            if want is not None:
                got = getattr(pages, name).transpose(1, 2).reshape(want.shape)
                assert torch.equal(got, want), name


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hd", [64, 128])
def test_cache_write_hands_nan_on(mode, hd):
    """A row with a NaN in any place reads back as NaN (16-bit rows: in that place),
    and so does what attends to it; the rows beside it are what they are without."""
    P = _api()
    g = _gen(hd)
    T, nkv = 200, 2
    k, v = (torch.randn(T, nkv, hd, generator=g, device="cuda") for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    clean, pages = (P.KVPages.empty(mode, 4, 64, nkv, hd, "cuda") for _ in range(2))
    P.paged_rope_kv(None, k, v, None, None, clean, table, lens, _cu([T]))
    at = (torch.arange(0, T, 3, device="cuda"), torch.arange(0, T, 3, device="cuda") % nkv)
    place = torch.arange(len(at[0]), device="cuda") % hd
    k[(*at, place)], v[(*at, hd - 1 - place)] = math.nan, math.nan
    P.paged_rope_kv(None, k, v, None, None, pages, table, lens, _cu([T]))
    for which, x in (("k", k), ("v", v)):
        got, was = (_values(t, which).transpose(1, 2).reshape(256, nkv, hd)[:T] for t in (pages, clean))
        want = x.isnan() if mode in ("fp16", "bf16") else x.isnan().any(-1, keepdim=True).expand_as(x)
        assert torch.equal(got.isnan(), want), which
        assert torch.equal(got[~want], was[~want]), which
    q = torch.randn(1, 2, hd, generator=g, device="cuda")
    assert P.paged_attention(q, pages, table, lens).isnan().all()


@gpu
@pytest.mark.parametrize("mode", ["int8", "2bit", "2bit_asym"])
def test_cache_write_beside_kv_quantize(mode):
    """How far a paged row is from the contiguous cache's.  The scale is a product
    with a rounded reciprocal for a quotient: three roundings, 3 * 2^-24 of itself.
    A code is off by at most one, and only where the value's place, of at most
    128 steps, is within 128 * 8 * 2^-24 of a border between two (the scales' 3,
    the quotients' 2, the sum's and the span's)."""
    P = _api()
    from polarflash_b200.kv_cache import kv_quantize

    T, nkv, hd = 4096, 2, 128
    k = torch.randn(T, nkv, hd, generator=_gen(3), device="cuda")
    k *= torch.exp2(torch.randint(-20, 20, (T, nkv, 1), generator=_gen(4), device="cuda").float())
    k[:512] = (k[:512] * 64).round() / 64  # many values that are equal parts of the largest
    pages = P.KVPages.empty(mode, T // 64, 64, nkv, hd, "cuda")
    table = torch.arange(T // 64, dtype=torch.int32, device="cuda")[None]
    P.paged_rope_kv(None, k, k, None, None, pages, table, torch.tensor([T], dtype=torch.int32, device="cuda"), _cu([T]))
    c, s, z = kv_quantize(k, mode)
    row = lambda t: t.transpose(1, 2).reshape(T, nkv, -1)  # noqa: E731
    mine, scale = row(pages.k), row(pages.k_scales[..., None])
    assert ((scale.double() / s.double() - 1).abs() <= 3.01 * 2.0 ** -24).all()
    x = k.double()
    if mode == "int8":
        place, border = x / s.double(), 0.5
    else:
        codes = lambda t: torch.stack([(t >> sh & 3) for sh in (6, 4, 2, 0)], -1).flatten(-2)  # noqa: E731
        c, mine = codes(c), codes(mine)
        place, border = (x / s.double() + 2, 0.0) if mode == "2bit" else ((x - z.double()) / s.double(), 0.5)
        if z is not None:
            assert torch.equal(row(pages.k_zeros[..., None]), z)
    off = (c.int() - mine.int()).abs()
    assert int(off.max()) <= 1
    near = ((place - border) - (place - border).round()).abs() <= 128 * 8 * 2.0 ** -24
    assert (near | (off == 0)).all()
    assert int((off > 0).sum()) < 0.001 * off.numel()


@gpu
def test_cache_write_forms():
    """One token per sequence without cu_seqlens; no rotation; no queries; q
    rotated in place; nothing to do; many sequences (the search for a row's
    sequence takes several steps)."""
    P = _api()
    g = _gen(0)
    B, nh, nkv, hd, page = 1500, 4, 2, 64, 16
    pages = P.KVPages.empty("bf16", B, page, nkv, hd, "cuda")
    table = torch.randperm(B, generator=g, device="cuda").to(torch.int32)[:, None].contiguous()
    lens = torch.randint(1, page + 1, (B,), generator=g, device="cuda").to(torch.int32)
    q, k, v = (torch.randn(B, h, hd, generator=g, device="cuda") for h in (nh, nkv, nkv))
    ang = torch.rand(B, hd // 2, generator=g, device="cuda")
    seq = torch.arange(B, device="cuda")
    rows = lambda t: t[table[:, 0].long(), :, lens.long() - 1]  # noqa: E731
    for cu in (None, torch.arange(B + 1, dtype=torch.int32, device="cuda")):
        pages.k.zero_(), pages.v.zero_()
        qo, ko, vo = P.paged_rope_kv(q, k, v, None, None, pages, table, lens, cu)
        assert ko is None and vo is None and torch.equal(qo, q)
        assert torch.equal(rows(pages.k), k.bfloat16()) and torch.equal(rows(pages.v), v.bfloat16())
        assert int((pages.k != 0).any(-1).sum()) == B * nkv  # nothing else was written
    q2 = q.clone()
    a = P.paged_rope_kv(q, k, v, ang.cos(), ang.sin(), pages, table, lens)[0]
    b = P.paged_rope_kv(q2, k, v, ang.cos(), ang.sin(), pages, table, lens, q_out=q2)[0]
    assert b is q2 and torch.equal(a, q2) and not torch.equal(a, q)
    pages.v.zero_()
    assert P.paged_rope_kv(None, k, v, None, None, pages, table, lens) == (None, None, None)
    assert torch.equal(rows(pages.v), v.bfloat16())
    e = P.paged_rope_kv(q[:0], k[:0], v[:0], None, None, pages, table[:0], lens[:0])[0]
    assert e.shape == (0, nh, hd)
    # ragged: 700 sequences, most of them empty
    new = (torch.rand(700, generator=g, device="cuda") > 0.7).int() * 2
    new[-1] = 2
    cu = torch.cat((new.new_zeros(1), new.cumsum(0).int()))
    T = int(cu[-1])
    pages.k.zero_()
    P.paged_rope_kv(None, k[:T], v[:T], None, None, pages, table[:700], new, cu)
    owner = torch.repeat_interleave(seq[:700], new.long())
    place = torch.arange(T, device="cuda") - cu.long()[owner]
    assert torch.equal(pages.k[table[owner, 0].long(), :, place], k[:T].bfloat16())


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hd,nh,odt", [(128, 6, torch.bfloat16), (64, 7, torch.float32)])
def test_cache_write_of_many_rows(mode, hd, nh, odt):
    """Calls large enough for several rows per warp, ten and eleven rows a token:
    the same bits as token by token."""
    P = _api()
    g = _gen(hd)
    nkv, page, lens = 2, 32, [900, 1, 700, 333]
    T, N = sum(lens), sum(-(-n // 32) for n in lens)
    table = _block_table(lens, page, N, g)
    lens_t, cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), _cu(lens)
    q, k, v = (torch.randn(T, h, hd, generator=g, device="cuda") for h in (nh, nkv, nkv))
    ang = torch.rand(T, hd // 2, generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    big, small = (P.KVPages.empty(mode, N, page, nkv, hd, "cuda") for _ in range(2))
    want = []
    at = 0
    for b, n in enumerate(lens):  # at most 100 tokens of one sequence: a row per warp
        for i in range(0, n, 100):
            m = min(100, n - i)
            sl = slice(at + i, at + i + m)
            want.append(P.paged_rope_kv(q[sl], k[sl], v[sl], cos[sl], sin[sl], small, table[b:b + 1].contiguous(),
                                        torch.tensor([i + m], dtype=torch.int32, device="cuda"), _cu([m]),
                                        out_dtype=odt, return_kv=True))
        at += n
    got = P.paged_rope_kv(q, k, v, cos, sin, big, table, lens_t, cu, out_dtype=odt, return_kv=True)
    for i in range(3):
        assert torch.equal(got[i], torch.cat([w[i] for w in want]))
    for name in ("k", "v", "k_scales", "v_scales", "k_zeros", "v_zeros"):
        if getattr(big, name) is not None:
            assert torch.equal(getattr(big, name), getattr(small, name)), name
    # and the formulas, for the keys of the last sequence
    x = k[-lens[3]:]
    c, s = cos[-lens[3]:, None], sin[-lens[3]:, None]
    x = torch.cat((x[..., : hd // 2] * c - x[..., hd // 2:] * s, x[..., : hd // 2] * s + x[..., hd // 2:] * c), -1)
    pos = torch.arange(lens[3], device="cuda")
    held = big.k[table[3].long()[pos // page], :, pos % page]
    assert torch.equal(held, x.to(held.dtype) if mode in ("fp16", "bf16") else _quantize(x, mode)[0])


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("nh,nkv,hd,page,dt", [
    (8, 2, 128, 16, torch.float32), (4, 4, 64, 64, torch.float32), (16, 2, 128, 32, torch.bfloat16),
    (6, 2, 64, 128, torch.float16), (7, 1, 128, 256, torch.float32), (24, 1, 64, 16, torch.bfloat16), (40, 8, 128, 64, torch.float32)])
def test_paged_attention(mode, nh, nkv, hd, page, dt):
    """Lengths around tile and page ends, none and one, longer than the table;
    NaN and infinity in slots and pages that no sequence sees; one page that
    is not of the cache."""
    P = _api()
    g = _gen(nh * hd + page)
    lens = [0, 1, 2, 15, 16, 17, page - 1, page, page + 1, 63, 64, 65, 300, 1000, 0, 257]
    N = sum(-(-n // page) for n in lens) + 5
    pages = _filled(P, mode, N, page, nkv, hd, g)
    table = _block_table(lens, page, N, g)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lens_t[12] = 300 if page > 64 else table.shape[1] * page + 1000  # cut at the table's end, whose pages are -1 there
    lens_t[14] = -3
    table[13, 1] = N + 7
    used = torch.zeros(N, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens_t.tolist()):
        for j in range(min(-(-n // page), table.shape[1])):
            if 0 <= int(table[b, j]) < N:
                used[int(table[b, j]), : min(page, n - j * page)] = True
    hole = ~used[:, None].expand(N, nkv, page)
    if mode in ("fp16", "bf16"):
        pages.k[hole], pages.v[hole] = math.nan, math.inf
    else:
        pages.k_scales[hole], pages.v_scales[hole] = math.nan, math.inf
        if mode == "2bit_asym":
            pages.k_zeros[hole], pages.v_zeros[hole] = math.inf, math.nan
    q = torch.randn(len(lens), nh, hd, generator=g, device="cuda").to(dt)
    for scale in (None, 0.03):
        got = P.paged_attention(q, pages, table, lens_t, scale=scale)
        want, mag = _attend64(pages, q, table, lens_t.tolist(), scale or hd ** -0.5)
        _near(got, want, mag, 1.6e-5)
        assert (got[[0, 14]] == 0).all()
    same = q.clone()
    assert torch.equal(P.paged_attention(same, pages, table, lens_t, scale=0.03, out=same), got)  # in place


@gpu
def test_paged_attention_extremes():
    """Scores far apart and large, values of very different sizes, all rows
    zero, and a long context whose late rows weigh most."""
    P = _api()
    g = _gen(3)
    for mode in MODES:
        pages = _filled(P, mode, 40, 64, 1, 128, g, spread=3.0 if mode != "fp16" else 1.0)
        lens = torch.tensor([2500, 2500, 1, 70], dtype=torch.int32, device="cuda")
        table = torch.stack([torch.randperm(40, generator=g, device="cuda") for _ in range(4)]).to(torch.int32)
        q = torch.randn(4, 4, 128, generator=g, device="cuda")
        want, mag = _attend64(pages, q, table, lens.tolist(), 0.05)
        _near(P.paged_attention(q, pages, table, lens, scale=0.05), want, mag, 1.6e-5)
        big = q * 50  # scores up to about 10^4: the weight of the largest is 1 or close to it
        sc = 0.05 * 50 * 6 * 128 * 3  # sum |q k| scale, at most
        want, mag = _attend64(pages, big, table, lens.tolist(), 0.05)
        _near(P.paged_attention(big, pages, table, lens, scale=0.05), want, mag, sc * 2.0 ** -21)
        z = P.KVPages.empty(mode, 2, 16, 1, 64, "cuda")
        got = P.paged_attention(q[:1, :, :64].contiguous(), z, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"),
                                torch.tensor([20], dtype=torch.int32, device="cuda"))
        assert (got == 0).all()


@gpu
@pytest.mark.parametrize("B,n,mode", [(1, 33000, "int8"), (300, 40, "2bit"), (3, 5000, "bf16")])
def test_paged_attention_split(B, n, mode):
    """Long and many: the positions of one sequence are shared by many blocks,
    and one block serves many sequences."""
    P = _api()
    g = _gen(B)
    lens = [max(0, n - 7 * i) for i in range(B)]
    N = sum(-(-m // 64) for m in lens)
    pages = _filled(P, mode, N, 64, 2, 128, g, 0.3)
    table = _block_table(lens, 64, N, g)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(B, 8, 128, generator=g, device="cuda")
    want, mag = _attend64(pages, q, table, lens, 128 ** -0.5)
    got = P.paged_attention(q, pages, table, lens_t)
    _near(got, want, mag, 1.6e-5)
    assert torch.equal(got, P.paged_attention(q, pages, table, lens_t))  # the same sums in the same order


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_paged_attention_long_sums(mode):
    """Many keys of like weight: the values nearly cancel, and what fp32 sums of
    n terms leave of the result, sqrt(n) 2^-24 of sum p |v| here (n = 20000, sums
    split over at least 32 warps), is below 1e-5 of its norm."""
    P = _api()
    g = _gen(11)
    pages = _filled(P, mode, 320, 64, 2, 128, g, spread=0.0)
    lens = torch.tensor([20000], dtype=torch.int32, device="cuda")
    table = torch.randperm(320, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    q = 0.3 * torch.randn(1, 16, 128, generator=g, device="cuda")
    want, mag = _attend64(pages, q, table, lens.tolist(), 128 ** -0.5)
    got = P.paged_attention(q, pages, table, lens)
    assert float((got.double() - want).norm() / want.norm()) < 1e-5


@gpu
@pytest.mark.parametrize("nh", [4, 8])
def test_paged_attention_over_the_range_of_bf16(nh):
    """bf16 pages with values up to bf16's largest and down to 2^-90."""
    P = _api()
    g = _gen(nh)
    lens = [1, 50, 3000, 20000]
    pages = _filled(P, "bf16", 400, 64, 1, 128, g, spread=0.0)
    unit = (pages.v.float().clamp(-3, 3) / 3).double()
    table = _block_table(lens, 64, 400, g)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(4, nh, 128, generator=g, device="cuda")
    for size in (0.9 * torch.finfo(torch.bfloat16).max, 2.0 ** 115, 2.0 ** -90):
        for flat in (False, True):  # flat: one sign, so that the sums grow with the length
            pages.v.copy_((unit.abs() if flat else unit) * size)
            for scale in (0.0, 128 ** -0.5):
                want, mag = _attend64(pages, q, table, lens, scale)
                _near(P.paged_attention(q, pages, table, lens_t, scale=scale), want, mag, 1.6e-5)


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("nh,hd", [(4, 128), (8, 64)])
def test_paged_attention_hands_nan_on(mode, nh, hd):
    """A NaN in a query head, or in a key that a sequence sees, makes NaN of the
    heads that meet it, whichever warp and block has it, and of no others."""
    P = _api()
    g = _gen(nh)
    lens = [1, 17, 130, 9000, 0]
    pages = _filled(P, mode, 200, 64, 2, hd, g, spread=0.3)
    table = _block_table(lens, 64, 200, g)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(5, nh, hd, generator=g, device="cuda")
    clean = P.paged_attention(q, pages, table, lens_t)
    bad = q.clone()
    bad[:, 1, 3] = math.nan
    got = P.paged_attention(bad, pages, table, lens_t)
    assert got[:4, 1].isnan().all() and (got[4] == 0).all()
    keep = [h for h in range(nh) if h != 1]
    assert torch.equal(got[:, keep], clean[:, keep])
    for b, pos in ((0, 0), (1, 0), (1, 16), (2, 129), (3, 0), (3, 4444), (3, 8999)):
        page, slot = int(table[b, pos // 64]), pos % 64
        rows = pages.k if mode in ("fp16", "bf16") else pages.k_scales
        was = rows[page, 1, slot].clone()
        rows[page, 1, slot] = math.nan
        got = P.paged_attention(q, pages, table, lens_t)
        rows[page, 1, slot] = was
        want = clean.clone()
        want[b, nh // 2:] = math.nan
        assert torch.equal(got.isnan(), want.isnan()), (b, pos)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), (b, pos)


@gpu
@pytest.mark.parametrize("nh", [4, 8])
def test_paged_attention_of_rows_that_hardly_vary(nh):
    """2bit_asym rows whose zero is up to 2^130 times their scale (a constant row's
    scale is 1e-8, whatever its value is), beside ordinary ones."""
    P = _api()
    g = _gen(nh)
    lens = [1, 40, 700, 5000]
    pages = _filled(P, "2bit_asym", 120, 64, 1, 128, g, spread=0.0)
    table = _block_table(lens, 64, 120, g)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(4, nh, 128, generator=g, device="cuda")
    zeros, scales = pages.v_zeros.clone(), pages.v_scales.clone()
    for size in (1.0, 1e10, 1e30, -1e30):
        for every in (1, 3):
            pages.v_zeros.copy_(zeros), pages.v_scales.copy_(scales)
            pages.v_zeros[:, :, ::every], pages.v_scales[:, :, ::every] = size, 1e-8
            want, mag = _attend64(pages, q, table, lens, 128 ** -0.5)
            _near(P.paged_attention(q, pages, table, lens_t), want, mag, 1.6e-5)


# ---- prompts ------------------------------------------------------------------------
def _prompt64(q, k, v, cq, ck, scale):
    out, mag = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    G = q.shape[1] // k.shape[1]
    for b in range(len(cq) - 1):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(q.shape[1]):
            s = q[cq[b]:cq[b + 1], h].double() @ k[ck[b]:ck[b + 1], h // G].double().T * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            vv = v[ck[b]:ck[b + 1], h // G].double()
            out[cq[b]:cq[b + 1], h], mag[cq[b]:cq[b + 1], h] = p @ vv, p @ vv.abs()
    return out, mag


def _cu(lens):
    return torch.tensor([0] + list(lens), device="cuda").cumsum(0).to(torch.int32)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", [
    (4, 4, 128, [1], [0]), (4, 2, 128, [127], [0]), (2, 1, 64, [128], [0]), (4, 2, 64, [129, 1, 255, 256, 257], [0] * 5),
    (8, 2, 128, [300, 0, 5, 513], [0] * 4), (6, 2, 128, [33, 1, 200, 0, 64], [100, 1000, 0, 7, 129]),
    (4, 1, 40, [70, 300], [13, 0]), (2, 2, 8, [150], [50]), (3, 1, 96, [260, 31], [0, 500]),
    (2, 1, 128, [64, 300, 20], [-30, -200, -20])])
def test_prompt_attention(dt, nh, nkv, hd, lens, past):
    """Lengths around the tiles' ends, empty sequences, cached prefixes, more
    queries than keys (rows that see none), every kind of head size, rows
    behind the last sequence left as they were, and strided rows."""
    P = _api()
    g = _gen(sum(lens) + hd)
    cq, ck = _cu(lens), _cu([a + b for a, b in zip(lens, past)])
    T, TK = int(cq[-1]) + 3, int(ck[-1]) + 2
    q = torch.randn(T, nh, hd, generator=g, device="cuda").to(dt)
    kv = torch.randn(TK, 2 * nkv * hd + 8, generator=g, device="cuda").to(dt)
    k, v = (kv[:, i * nkv * hd:(i + 1) * nkv * hd].unflatten(1, (nkv, hd)) for i in range(2))
    v[int(ck[-1]):] = math.nan  # behind the last sequence
    k[int(ck[-1]):] = math.nan
    out = torch.full((T, nh * hd + 16), 7.0, dtype=dt, device="cuda")
    view = out[:, : nh * hd].unflatten(1, (nh, hd))
    for scale in (None, 0.2):
        P.prompt_attention(q, k, v, cq, ck, scale=scale, out=view)
        n = int(cq[-1])
        want, mag = _prompt64(q, k, v, cq.tolist(), ck.tolist(), scale or hd ** -0.5)
        e = HALF_STEP[dt]
        off = (view[:n].double() - want[:n]).abs()
        bound = (2.5 * e + 1.6e-5) * mag[:n] + (2.0 ** -24 * TK if dt == torch.float16 else 1e-30)
        assert (off <= bound).all(), float((off / bound).max())
        assert (out[n:] == 7).all() and (out[:, nh * hd:] == 7).all()


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_prompt_attention_row_norms(dt, hd):
    """Row by row, normwise: a rounding by half a step e is e / sqrt(6) of its value
    in the root of the mean square (an error even in -e..e, over values even in a
    binade).  The weights and the output are rounded once each, and with values of
    random sign both count alike: 0.58 e, over 4 heads of as many dimensions and at
    least 64 keys of like weight; below e.  A key too many or too few among n is
    1 / sqrt(n) of a row's norm: six times the bound for bf16 at 2000 keys."""
    P = _api()
    g = _gen(hd)
    lens, past = [2000, 700, 128], [0, 300, 129]
    cq, ck = _cu(lens), _cu([a + b for a, b in zip(lens, past)])
    q = (0.3 * torch.randn(sum(lens), 4, hd, generator=g, device="cuda")).to(dt)
    k, v = (torch.randn(int(ck[-1]), 2, hd, generator=g, device="cuda").to(dt) for _ in range(2))
    got = P.prompt_attention(q, k, v, cq, ck)
    want, _ = _prompt64(q, k, v, cq.tolist(), ck.tolist(), hd ** -0.5)
    off = (got.double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    keys = torch.cat([torch.arange(p + 1, p + n + 1, device="cuda") for n, p in zip(lens, past)])
    assert float(off[keys >= 64].max()) < HALF_STEP[dt]


@gpu
def test_prompt_attention_of_many_sequences():
    """100 sequences, some of them empty, of up to 150 queries; keys for some
    only; and no key at all."""
    P = _api()
    g = _gen(8)
    lens = [(37 * i) % 150 if i % 9 else 0 for i in range(100)]
    keys = [n + (i % 40) if i % 7 else 0 for i, n in enumerate(lens)]
    cq, ck = _cu(lens), _cu(keys)
    q = torch.randn(sum(lens), 6, 64, generator=g, device="cuda").half()
    k, v = (torch.randn(sum(keys), 2, 64, generator=g, device="cuda").half() for _ in range(2))
    got = P.prompt_attention(q, k, v, cq, ck)
    want, mag = _prompt64(q, k, v, cq.tolist(), ck.tolist(), 0.125)
    assert ((got.double() - want).abs() <= (2.5 * 2.0 ** -11 + 1.6e-5) * mag + 2.0 ** -24 * 200).all()
    none = P.prompt_attention(q, k[:0], v[:0], cq, torch.zeros_like(cq))
    assert (none == 0).all()
    assert P.prompt_attention(q[:0], k, v, torch.zeros_like(cq), ck).shape == (0, 6, 64)
    from polarflash_b200.serving import check_serving_status

    check_serving_status("cuda")  # no wait has given up


@gpu
def test_prompt_attention_keeps_sequences_apart():
    """NaN and infinity in one sequence's k and v do not reach another's rows,
    in a key's later place not through k, and large scores do not overflow."""
    P = _api()
    g = _gen(5)
    cu = _cu([100, 200, 77])
    q, k, v = (torch.randn(377, h, 128, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    clean = P.prompt_attention(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    v2[100:300], k2[100:300] = math.nan, math.inf
    got = P.prompt_attention(q, k2, v2, cu)
    for s in (slice(0, 100), slice(300, 377)):
        assert torch.equal(got[s], clean[s])
    k3 = k.clone()
    k3[250:300] = math.nan  # rows 100..249 do not see these keys
    assert torch.equal(P.prompt_attention(q, k3, v, cu)[100:250], clean[100:250])
    v3 = v.clone()
    v3[250:255], v3[255:300, 1, :50] = math.nan, math.inf  # nor these, which share tiles with them
    got = P.prompt_attention(q, k3, v3, cu)
    want, mag = _prompt64(q, k, v, cu.tolist(), cu.tolist(), 128 ** -0.5)
    off = (got[100:250].double() - want[100:250]).abs()
    assert (off <= (2.5 * 2.0 ** -8 + 1.6e-5) * mag[100:250]).all()
    for s in (slice(0, 100), slice(300, 377)):
        assert torch.equal(got[s], clean[s])
    assert torch.isnan(got[250:300]).all()  # (k3 is NaN there too)
    assert torch.isnan(P.prompt_attention(q, k, v3, cu)[250:300]).all()
    few = P.prompt_attention(q[100:120], k[100:110], v3[250:260], _cu([20]), _cu([10]))
    assert (few[:10] == 0).all() and torch.isnan(few[10:]).all()  # rows without a key: 0, whatever v holds
    big = P.prompt_attention((q * 100).bfloat16(), (k * 100).bfloat16(), v, cu)
    assert torch.isfinite(big).all()
    want, mag = _prompt64((q * 100).bfloat16(), (k * 100).bfloat16(), v, cu.tolist(), cu.tolist(), 128 ** -0.5)
    # scores reach 10^5 here: fp32 leaves 2^-24 * 10^5 * 8 roundings = 0.05 of them, a weight's relative error
    off = (big.double() - want).abs()
    assert (off <= (2.5 * 2.0 ** -8 + 0.1) * mag).all()


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_weighs_hidden_keys_nothing(dt, hd):
    """Values near the type's largest at keys that a row does not see, and at a
    key whose score lies hundreds below the maximum, change nothing: their weight
    is 0, in every place of a tile."""
    P = _api()
    g = _gen(hd)
    n = 300
    cu = _cu([n])
    q, k, v = (torch.randn(n, h, hd, generator=g, device="cuda").to(dt) for h in (4, 2, 2))
    big = torch.finfo(dt).max * 0.9
    clean = P.prompt_attention(q, k, v, cu)
    for first in (100, 128, 145, 200, 256, 272):
        for j in range(16):
            late = v.clone()
            late[first + j::16] = big
            got = P.prompt_attention(q, k, late, cu)
            assert torch.equal(got[:first], clean[:first]), (first, j)
    # one direction, along which key `at` scores 40 * 8 * sqrt(hd) / sqrt(hd) = 320 and more below every other
    q = torch.full((n, 4, hd), 8.0, dtype=dt, device="cuda")
    for at in (0, 1, 2, 17, 130, 144):
        low = torch.randn(n, 2, hd, generator=g, device="cuda").to(dt).abs()
        low[at] = -40.0
        v0, v1 = v.clone(), v.clone()
        v0[at], v1[at] = 0.0, big
        assert torch.equal(P.prompt_attention(q, low, v1, cu)[at + 1:], P.prompt_attention(q, low, v0, cu)[at + 1:]), at


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_hands_nan_on(dt, hd):
    """A NaN in k makes NaN of every value of the rows that see it, wherever in a
    tile it stands and whatever scores follow it, and of no other row."""
    P = _api()
    n = 300
    cu = _cu([n])
    q, k, v = (torch.randn(n, h, hd, generator=_gen(hd), device="cuda").to(dt) for h in (4, 2, 2))
    k[256:] *= 30  # larger scores later: what was summed up before is scaled down
    clean = P.prompt_attention(q, k, v, cu)
    for at in (*range(17), 128, 129, 145, 270):
        bad = k.clone()
        bad[at, 1, hd // 2] = math.nan
        got = P.prompt_attention(q, bad, v, cu)
        assert got[at:, 2:].isnan().all(), at
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[:, :2], clean[:, :2])


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_prompt_attention_of_infinite_scores(dt):
    """Scores of -inf weigh nothing beside finite ones, before and behind them; a
    row with nothing else is 0 / 0, NaN, as the definition has it, while a row
    without keys is zeros."""
    P = _api()
    g = _gen(2)
    n, hd = 200, 64
    cu = _cu([n])
    q = torch.rand(n, 2, hd, generator=g, device="cuda").to(dt) + 0.1
    k, v = (torch.randn(n, 1, hd, generator=g, device="cuda").to(dt) for _ in range(2))
    for cut in (1, 17, 128, 150):
        low = k.clone()
        low[:cut] = -math.inf
        got = P.prompt_attention(q, low, v, cu)
        assert got[:cut].isnan().all(), cut
        # the same rows over the other keys alone
        rest = P.prompt_attention(q[cut:], k[cut:], v[cut:], _cu([n - cut]))
        e = HALF_STEP[dt]
        _, mag = _prompt64(q[cut:], k[cut:], v[cut:], [0, n - cut], [0, n - cut], hd ** -0.5)
        # each of the two is off by no more than the bound of a prompt
        assert ((got[cut:].double() - rest.double()).abs() <= 2 * ((2.5 * e + 1.6e-5) * mag + 2.0 ** -24 * n)).all(), cut
    few = P.prompt_attention(q[:20], low[:10], v[:10], _cu([20]), _cu([10]))
    assert (few[:10] == 0).all() and few[10:].isnan().all()


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_over_the_range_of_bf16(hd):
    """Values up to bf16's largest and down to 2^-90, for flat weights and for
    scores that rise along the keys."""
    P = _api()
    g = _gen(hd)
    lens = [1400, 3, 130]
    cu, T = _cu(lens), sum(lens)
    q, k, v = (torch.randn(T, h, hd, generator=g, device="cuda").bfloat16() for h in (2, 1, 1))
    q = q.abs()
    rise = (k.abs() * torch.linspace(0.1, 3, T, device="cuda")[:, None, None]).bfloat16()
    v = v.clamp(-3, 3) / 3
    for keys in (k, rise):
        for size in (0.9 * torch.finfo(torch.bfloat16).max, 2.0 ** 115, 2.0 ** -90):
            vv = (v.double() * size).bfloat16()
            got = P.prompt_attention(q, keys, vv, cu)
            want, mag = _prompt64(q, keys, vv, cu.tolist(), cu.tolist(), hd ** -0.5)
            assert ((got.double() - want).abs() <= (2.5 * HALF_STEP[torch.bfloat16] + 1.6e-5) * mag).all(), size


# ---- the draw ---------------------------------------------------------------------
def _draw64(logits, u, t, k, p, m):
    """One row, in Python's and torch's fp64, entry by entry."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = float(x.max())
    if top == -math.inf:
        return -1
    if not t > 0:
        return int((x == top).nonzero()[0])
    w = torch.exp(torch.where(x == top, 0.0, (x - top) / t))
    order = torch.sort(x, descending=True, stable=True).indices
    if k > 0:
        order = order[:k]
    if not p >= 1:
        ws = w[order]
        before = torch.cat((ws.new_zeros(1), ws.cumsum(0)[:-1]))
        keep = before < p * float(ws.sum())
        keep[0] = True
        order = order[keep]
    order = order[w[order] >= min(m, 1.0)]
    kept = torch.zeros_like(w)
    kept[order] = w[order]
    c = kept.cumsum(0)
    over = (c > u * float(c[-1])).nonzero()
    return int(over[0]) if len(over) else int((kept > 0).nonzero()[-1])


def _check_draw(P, logits, u, t=1.0, k=0, p=1.0, m=0.0):
    R = logits.shape[0]
    got = P.sample_logits(logits, u, temperature=t, top_k=k, top_p=p, min_p=m).tolist()
    at = lambda x, i: (x[i].item() if isinstance(x, torch.Tensor) else float(torch.tensor(x, dtype=torch.float32)) if isinstance(x, float) else x)  # noqa: E731
    lg, uu = logits.cpu(), u.cpu()
    for i in range(R):
        want = _draw64(lg[i], uu[i].item(), at(t, i), at(k, i), at(p, i), at(m, i))
        assert got[i] == want, (i, got[i], want)


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 384, 1023, 4097, 32001, 128256])
def test_draw_matches_the_definition(dt, V):
    P = _api()
    g = _gen(V)
    R = 12
    wide = (3 * torch.randn(R, V + 5, generator=g, device="cuda")).to(dt)
    logits = wide[:, :V] if V % 2 else wide[:, 3:V + 3]  # strided rows, odd starts
    u = torch.rand(R, generator=g, device="cuda")
    _check_draw(P, logits, u)
    _check_draw(P, logits, u, t=0.7, p=0.9)
    _check_draw(P, logits, u, t=1.3, k=5)
    _check_draw(P, logits, u, t=0.9, k=50, p=0.8, m=0.02)
    _check_draw(P, logits, u, t=2.0, m=0.1)
    _check_draw(P, logits, u, t=0.0)
    r = lambda: torch.rand(R, generator=g, device="cuda")  # noqa: E731
    _check_draw(P, logits, u, t=2 * r() * (r() > 0.2), k=(r() * 2 * V).int(), p=1.2 * r(), m=0.2 * r())


@gpu
def test_draw_at_the_largest_vocabulary():
    """360000 entries: slices of 45000; equal logits (sums near 2^63) and spread ones."""
    P = _api()
    V = 360000
    u = torch.tensor([0.1, 0.5, 0.999], device="cuda")
    flat = torch.zeros(3, V, device="cuda")
    wide = 2 * torch.randn(3, V, generator=_gen(2), device="cuda")
    for kw in (dict(), dict(k=V - 1), dict(k=V - 1, p=0.75), dict(p=0.3), dict(k=70000, p=0.9, m=0.001)):
        _check_draw(P, flat, u, **kw)
        _check_draw(P, wide, u, **kw)


@gpu
def test_draw_of_equal_and_missing_logits():
    """Ties (top-k and top-p cut inside them, the lowest index first), zeros of
    both signs, NaN, infinities, rows of -inf, and the ends of u."""
    P = _api()
    V = 5000
    dev = dict(device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24], **dev)
    R = len(u)
    flat = torch.zeros(R, V, **dev)
    flat[:, 1::2] = -0.0
    for kw in (dict(), dict(k=7), dict(p=0.5), dict(k=1000, p=0.25), dict(k=3, p=0.4), dict(p=0.0), dict(p=-1.0), dict(k=V),
               dict(k=V + 9), dict(k=2 ** 32 + 5), dict(k=-7), dict(m=1.0), dict(m=3.0), dict(t=0.0), dict(t=-1.0), dict(t=100.0)):
        _check_draw(P, flat, u, **kw)
    two = torch.full((R, V), -math.inf, **dev)
    two[:, 17], two[:, 4000] = 1.0, 1.0
    for kw in (dict(), dict(k=1), dict(k=2), dict(k=3), dict(p=0.5), dict(p=0.51), dict(t=0.0)):
        _check_draw(P, two, u, **kw)
    odd = torch.randn(R, V, generator=_gen(1), **dev)
    odd[:, ::3], odd[:, 1::7] = math.nan, -math.inf
    for kw in (dict(), dict(k=40, p=0.9), dict(t=0.0)):
        _check_draw(P, odd, u, **kw)
    odd[:, 99], odd[:, 2100] = math.inf, math.inf
    for kw in (dict(), dict(k=1), dict(k=9, p=0.3), dict(t=0.0), dict(m=0.5)):
        _check_draw(P, odd, u, **kw)
    none = torch.full((R, V), -math.inf, **dev)
    none[1:3] = math.nan
    for kw in (dict(), dict(t=0.0), dict(k=3, p=0.5)):
        assert P.sample_logits(none, u, temperature=kw.get("t", 1.0), top_k=kw.get("k", 0), top_p=kw.get("p", 1.0)).tolist() == [-1] * R
    over = torch.tensor([1.0, 2.0, math.inf], **dev)  # u outside [0, 1): the last kept token
    _check_draw(P, odd[:3], over, k=5)
    steps = torch.arange(V, 0, -1, **dev).float()[None].repeat(R, 1) * 2.0 ** -10  # many levels, few of weight
    for kw in (dict(t=0.01, p=0.99), dict(t=0.001, k=3), dict(t=50.0, p=0.37), dict(t=1e-6)):
        _check_draw(P, steps, u, **kw)
    far = torch.tensor([[-3e38, 3e38, 3e38, -3e38, 1.0]], **dev).repeat(R, 1)
    for kw in (dict(), dict(k=3), dict(p=0.6), dict(t=0.0)):
        _check_draw(P, far, u, **kw)


# ---- calls -------------------------------------------------------------------------
@gpu
def test_serving_ops_refuse():
    P = _api()
    dev = "cuda"
    pages = P.KVPages.empty("int8", 4, 16, 2, 64, dev)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    q, k = torch.zeros(2, 4, 64, device=dev), torch.zeros(2, 2, 64, device=dev)
    h = q.half()
    bad = [
        lambda: P.KVPages.empty("fp32", 4, 16, 2, 64, dev), lambda: P.KVPages.empty("int8", 4, 17, 2, 64, dev),
        lambda: P.KVPages.empty("int8", 4, 16, 2, 80, dev), lambda: P.KVPages.empty("int8", 0, 16, 2, 64, dev),
        lambda: P.KVPages("int8", pages.k, pages.v), lambda: P.KVPages("int8", pages.k, pages.v[:, :1], pages.k_scales, pages.v_scales),
        lambda: P.KVPages("2bit_asym", pages.k, pages.v, pages.k_scales, pages.v_scales),
        lambda: P.KVPages("int8", pages.k.cpu(), pages.v.cpu(), pages.k_scales, pages.v_scales),
        lambda: P.paged_attention(q.double(), pages, i32(2, 1), i32(2)), lambda: P.paged_attention(q[:, :3], pages, i32(2, 1), i32(2)),
        lambda: P.paged_attention(q, pages, i32(2, 1).long(), i32(2)), lambda: P.paged_attention(q, pages, i32(2, 1), i32(3)),
        lambda: P.paged_attention(q, pages, i32(2, 0), i32(2)), lambda: P.paged_attention(q.cpu(), pages, i32(2, 1), i32(2)),
        lambda: P.paged_attention(q, pages, i32(2, 1), i32(2), out=q.half()),
        lambda: P.paged_attention(q, pages, i32(2, 1), i32(2), workspace=torch.zeros(16, dtype=torch.uint8, device=dev)),
        lambda: P.paged_rope_kv(q, k, k.half(), None, None, pages, i32(2, 1), i32(2)),
        lambda: P.paged_rope_kv(q, k, k, q[:, 0, :32], None, pages, i32(2, 1), i32(2)),
        lambda: P.paged_rope_kv(q[:1], k, k, None, None, pages, i32(2, 1), i32(2)),
        lambda: P.paged_rope_kv(q, k, k, None, None, pages, i32(1, 1), i32(1)),
        lambda: P.paged_rope_kv(q, k, k, None, None, pages, i32(2, 1), i32(2), out_dtype=torch.int8),
        lambda: P.paged_rope_kv(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, None, None, pages, i32(2, 1), i32(2)),
        lambda: P.paged_rope_kv(None, k, k, None, None, pages, i32(2, 1), i32(2), q_out=q),
        lambda: P.prompt_attention(q, k, k, i32(2)), lambda: P.prompt_attention(q.half(), k.bfloat16(), k.bfloat16(), i32(2)),
        lambda: P.prompt_attention(q.half(), k[:1].half(), k[:1].half(), i32(2)),
        lambda: P.prompt_attention(q[:, :3].half(), k.half(), k.half(), i32(2)),
        lambda: P.prompt_attention(q.half()[..., :60], k.half()[..., :60], k.half()[..., :60], i32(2)),
        lambda: P.prompt_attention(q.half(), k.half(), k.half(), i32(2), i32(3)),
        lambda: P.prompt_attention(h, h, h, i32(2), out=h),
        lambda: P.sample_logits(q[0].double(), q[0, 0, :4]), lambda: P.sample_logits(q[0], q[0, 0, :3]),
        lambda: P.sample_logits(q[0].T, q[0, 0, :64]), lambda: P.sample_logits(q[0], q[0, 0, :4].double()),
        lambda: P.sample_logits(q[0], q[0, 0, :4], top_k=q[0, 0, :4]), lambda: P.sample_logits(q[0, :, :0], q[0, 0, :4]),
        lambda: P.sample_logits(q[0].cpu(), q[0, 0, :4].cpu()),
    ]
    launches = _lib.kernel_launches()
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    assert _lib.kernel_launches() == launches


@gpu
def test_serving_ops_at_once():
    """Calls on two streams at the same time, each with workspaces of its own, give
    what they give alone."""
    P = _api()
    g = _gen(4)
    sides = []
    for i in range(2):
        pages = _filled(P, MODES[2 + i], 200, 64, 2, 128, g, 0.3)
        lens = torch.tensor([3000 - 700 * i, 17, 900, 0, 4000], dtype=torch.int32, device="cuda")
        table = torch.stack([torch.randperm(200, generator=g, device="cuda")[:64] for _ in range(5)]).to(torch.int32)
        sides.append(dict(pages=pages, lens=lens, table=table, q=torch.randn(5, 16, 128, generator=g, device="cuda"),
                          p=[torch.randn(700 + 90 * i, h, 128, generator=g, device="cuda").half() for h in (8, 2, 2)],
                          cu=_cu([500, 200 + 90 * i]), logits=2 * torch.randn(9, 60000 + 7 * i, generator=g, device="cuda"),
                          u=torch.rand(9, generator=g, device="cuda")))

    def call(s):
        return (P.paged_attention(s["q"], s["pages"], s["table"], s["lens"]), P.prompt_attention(*s["p"], s["cu"]),
                P.sample_logits(s["logits"], s["u"], temperature=0.9, top_k=1000, top_p=0.9))

    want = [call(s) for s in sides]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(sides[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@gpu
def test_serving_ops_on_streams_and_in_graphs():
    """The four operators in a row, as a decode step runs them: on another
    stream, and captured once and replayed on new inputs, with a second graph
    over the same buffers between; each equal to the eager calls."""
    P = _api()
    g = _gen(9)
    B, nh, nkv, hd, V = 5, 8, 2, 128, 1000
    lens = torch.tensor([3, 64, 65, 200, 1], dtype=torch.int32, device="cuda")
    table = torch.randperm(40, generator=g, device="cuda").to(torch.int32).view(5, 8)
    head = torch.randn(nh * hd, V, generator=g, device="cuda") * 0.05
    ins = [[torch.randn(B, h, hd, generator=g, device="cuda") for h in (nh, nkv, nkv)] + [torch.rand(B, generator=g, device="cuda")]
           for _ in range(3)]
    ang = torch.rand(B, hd // 2, generator=g, device="cuda")
    cos, sin = ang.cos(), ang.sin()

    def step(pages, x, ws):
        q, k, v, u = x
        q, _, _ = P.paged_rope_kv(q, k, v, cos, sin, pages, table, lens)
        o = P.paged_attention(q, pages, table, lens, workspace=ws)
        p = P.prompt_attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), torch.arange(B + 1, dtype=torch.int32, device="cuda"))
        return o, p, P.sample_logits(o.flatten(1) @ head, u, temperature=0.8, top_k=50, top_p=0.9)

    fresh = lambda: _filled(P, "int8", 40, 64, nkv, hd, _gen(1))  # noqa: E731
    eager = fresh()
    want = [[t.clone() for t in step(eager, x, None)] for x in ins]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = fresh()
        got = [[t.clone() for t in step(other, x, None)] for x in ins]
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    pages, x = fresh(), [t.clone() for t in ins[0]]
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda").fill_(255)
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        step(pages, x, ws)
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                outs.append(step(pages, x, ws))
            graphs.append(gr)
    torch.cuda.current_stream().wait_stream(s)
    for i, new in enumerate(ins):
        for a, b in zip(x, new):
            a.copy_(b)
        graphs[i % 2].replay()
        for a, b in zip(outs[i % 2], want[i]):
            assert torch.equal(a, b), i
    torch.cuda.synchronize()


@gpu
def test_serving_ops_beyond_32_bits():
    """Rows whose offsets pass 2^31 elements and 2^32 bytes: pages at the end of a
    large cache, strided prompts and logits; each as over compact copies."""
    P = _api()
    g = _gen(12)
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    # pages: 256 slots of 8 heads of 128, 2^18 elements each; 8300 of them pass 2^31
    nh, nkv, hd, N = 16, 8, 128, 8300
    lens = [300, 5, 256]
    table, near = i32([[N - 1, 0], [N - 3, -1], [8192, -1]]), i32([[0, 1], [2, -1], [3, -1]])
    T = sum(lens)
    x = [torch.randn(T, h, hd, generator=g, device="cuda") for h in (nh, nkv, nkv)]
    q = torch.randn(3, nh, hd, generator=g, device="cuda")
    for mode in ("bf16", "int8"):
        far, small = (P.KVPages.empty(mode, n, 256, nkv, hd, "cuda") for n in (N, 4))
        for pages, t in ((far, table), (small, near)):
            P.paged_rope_kv(*x, None, None, pages, t, i32(lens), _cu(lens))
        for which in ("k", "v"):
            assert torch.equal(getattr(far, which)[table[:, 0].long()], getattr(small, which)[near[:, 0].long()])
        assert torch.equal(P.paged_attention(q, far, table, i32(lens)), P.paged_attention(q, small, near, i32(lens)))
        del far
    # rows 2^23 elements apart
    wide = torch.empty(300, 1 << 23, dtype=torch.bfloat16, device="cuda")
    parts = [torch.randn(300, h, hd, generator=g, device="cuda").bfloat16() for h in (nh, nkv, nkv, nh)]
    at, views = 0, []
    for p in parts:
        views.append(wide[:, at:at + p.shape[1] * hd].unflatten(1, (-1, hd)))
        views[-1].copy_(p)
        at += p.shape[1] * hd
    cu = _cu([130, 170])
    P.prompt_attention(*views[:3], cu, out=views[3])
    assert torch.equal(views[3], P.prompt_attention(*parts[:3], cu))
    small, other = (P.KVPages.empty("int8", 4, 256, nkv, hd, "cuda") for _ in range(2))
    a = P.paged_rope_kv(*views[:3], None, None, small, near, i32([130, 170, 0]), _cu([130, 170, 0]))[0]
    b = P.paged_rope_kv(*parts[:3], None, None, other, near, i32([130, 170, 0]), _cu([130, 170, 0]))[0]
    assert torch.equal(a, b) and torch.equal(small.k, other.k) and torch.equal(small.v, other.v)
    logits = wide[:, :5000].copy_(3 * torch.randn(300, 5000, generator=g, device="cuda"))
    u = torch.rand(300, generator=g, device="cuda")
    kw = dict(temperature=0.8, top_k=50, top_p=0.9)
    assert torch.equal(P.sample_logits(logits, u, **kw), P.sample_logits(logits.contiguous(), u, **kw))
