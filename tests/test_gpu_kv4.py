"""GPU tests of the 4-bit K/V cache and the attention over it, against the
float64 restatement in oracle/kv4_ref.py.

Tolerances. The cache's values are exact: codes, scales and zeros are those
of exact arithmetic, and a value read back is rounded once. Attention: the
output's rounding is at most 2^-8 of the value; p * scale enters the product
with 11 bits (2^-11 relative, at most 2^-11 * |v - centre| in the weighted
mean, so below 2^-10 of the largest |v|); everything else is f32. Hence
|got - want| <= 2^-8 |want| + 2^-10 max|v|."""

import math

import pytest
import torch

from oracle import kv4_ref as kr

pytestmark = pytest.mark.gpu
PAGE = 64


def rows_like(shape, seed, device):
    """K/V-like values: channels of unequal size, some shifted, some outliers."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    size = torch.exp(0.5 * torch.randn(shape[-2], shape[-1], generator=g))
    x = (x + 0.5 * torch.randn(shape[-2], shape[-1], generator=g)) * size
    return x.to(torch.bfloat16).to(device)


def make_cache(lens, kv_heads, group, device, spare=3, fill=0xFF, seed=0, max_pages=None):
    """Pages in random order; every byte that nothing writes is `fill` (0xFF: NaN pairs)."""
    import ltxb
    g = torch.Generator().manual_seed(seed)
    per = max(-(-max(lens) // PAGE), 1) if max_pages is None else max_pages
    n = len(lens) * per + spare
    block = ltxb.lib.ltxb_kv4_block_bytes(group)
    pages = torch.full((n, kv_heads, block), fill, dtype=torch.uint8, device=device)
    table = torch.randperm(n, generator=g)[:len(lens) * per].view(len(lens), per).to(torch.int32).to(device)
    return ltxb.KV4Cache.from_pages(pages, table, torch.tensor(lens, dtype=torch.int32, device=device), group=group)


def starts(counts, device):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return torch.tensor(s, dtype=torch.int32, device=device)


def filled(lens, kv_heads, group, device, seed=0, **kw):
    """A cache holding whole sequences, and their f64 values [len, heads, 128]."""
    cache = make_cache(lens, kv_heads, group, device, seed=seed, **kw)
    k = rows_like((sum(lens), kv_heads, 128), seed + 1, device)
    v = rows_like((sum(lens), kv_heads, 128), seed + 2, device)
    cache.append(k, v, row_start=starts(lens, device))
    kh, vh = kr.held(k.cpu(), group), kr.held(v.cpu(), group)
    return cache, list(kh.split(list(lens))), list(vh.split(list(lens)))


def check(got, want, vmax, note=""):
    got = got.double().cpu()
    err = (got - want).abs()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -10 * vmax
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert bool((err <= bound).all()), f"{note}: {worst:.2f} of the bound"


# ---------------------------------------------------------------------------
# writing and reading
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("lens,kv_heads", [([1], 1), ([64, 1, 65], 2), ([130, 7, 63, 200], 5), ([0, 3, 0], 3)])
def test_append_and_read_are_exact(cuda, lens, kv_heads, group):
    cache = make_cache(lens, kv_heads, group, cuda)
    n = sum(lens)
    k, v = rows_like((n, kv_heads, 128), 1, cuda), rows_like((n, kv_heads, 128), 2, cuda)
    rs = starts(lens, cuda)
    cache.append(k, v, row_start=rs)
    kf, vf = cache.read(n, row_start=rs, dtype=torch.float32)
    kb, vb = cache.read(n, row_start=rs)
    wk, wv = kr.held(k.cpu(), group), kr.held(v.cpu(), group)
    for f, b, w in ((kf, kb, wk), (vf, vb, wv)):
        assert torch.equal(f.cpu(), w.float())
        assert torch.equal(b.cpu(), w.float().to(torch.bfloat16))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_block_bytes_are_the_documented_ones(cuda, group):
    lens, heads = [70], 2
    cache = make_cache(lens, heads, group, cuda, fill=0)
    k, v = rows_like((70, heads, 128), 5, cuda), rows_like((70, heads, 128), 6, cuda)
    cache.append(k, v)
    kc, ks, kz = kr.quantise(k.cpu(), group)
    vc, vs, vz = kr.quantise(v.cpu(), group)
    table, pages = cache.page_table.cpu(), cache.pages.cpu()
    ng = 128 // group
    for t in (0, 1, 9, 30, 63, 64, 69):
        for h in range(heads):
            block = bytes(pages[int(table[0, t // PAGE]), h].tolist())
            for d in range(128):
                assert kr.k_code(block, t % PAGE, d) == int(kc[t, h, d])
                assert kr.v_code(block, t % PAGE, d) == int(vc[t, h, d])
            pairs = pages[int(table[0, t // PAGE]), h, 8192:].clone().view(torch.bfloat16).view(2, PAGE, ng, 2)
            for i, (s, z) in enumerate(((ks, kz), (vs, vz))):
                assert torch.equal(pairs[i, t % PAGE, :, 0].double(), s[t, h])
                assert torch.equal(pairs[i, t % PAGE, :, 1].double(), z[t, h])


def test_append_touches_only_its_tokens(cuda):
    """One token at a time, in the middle of a page: the bytes of all other tokens stay."""
    cache = make_cache([100, 37], 3, 64, cuda, fill=0x5A)
    k, v = rows_like((2, 3, 128), 1, cuda), rows_like((2, 3, 128), 2, cuda)
    before = cache.pages.clone()
    cache.append(k, v)
    changed = {tuple(x) for x in (cache.pages != before).nonzero()[:, :2].tolist()}
    table = cache.page_table.cpu()
    assert changed == {(int(table[0, 1]), h) for h in range(3)} | {(int(table[1, 0]), h) for h in range(3)}
    for b, t in ((0, 99), (1, 36)):
        for h in range(3):
            blk, old = cache.pages[int(table[b, t // PAGE]), h].cpu(), before[int(table[b, t // PAGE]), h].cpu()
            t %= PAGE
            mine = torch.zeros(blk.numel(), dtype=torch.bool)
            mine[64 * t:64 * t + 64] = True
            for g in range(8):
                o = 4096 + 512 * (t // 8) + 64 * g + 16 * ((t % 8) // 2) + 8 * (t % 2)
                mine[o:o + 8] = True
            for o in (8192, 8192 + 64 * 8):
                mine[o + 8 * t:o + 8 * t + 8] = True
            assert torch.equal(blk[~mine], old[~mine])


def test_strided_rows_and_padding_rows(cuda):
    """k and v as slices of a fused projection; rows before, between and behind the ranges are left alone."""
    heads, group = 4, 32
    fused = rows_like((20, 3 * heads, 128), 3, cuda)
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    cache = make_cache([9, 0, 70], heads, group, cuda)
    rs = torch.tensor([2, 7, 7, 15], dtype=torch.int32, device=cuda)
    cache.append(k, v, row_start=rs)
    out = tuple(torch.full((20, heads, 128), 7.0, device=cuda) for _ in range(2))
    cache.read(20, row_start=rs, dtype=torch.float32, out=out)
    for got, src in zip(out, (k, v)):
        got = got.cpu()
        assert torch.equal(got[2:15], kr.held(src.cpu(), group).float()[2:15])
        assert bool((got[:2] == 7).all()) and bool((got[15:] == 7).all())


def test_tokens_before_the_first_do_not_exist(cuda):
    """More rows than tokens: the first rows have no place and are skipped."""
    cache = make_cache([2, 5], 2, 128, cuda)
    k, v = rows_like((8, 2, 128), 1, cuda), rows_like((8, 2, 128), 2, cuda)
    cache.append(k, v)
    out = tuple(torch.full((8, 2, 128), 3.0, device=cuda) for _ in range(2))
    cache.read(8, dtype=torch.float32, out=out)
    want = kr.held(k.cpu(), 128).float()
    got = out[0].cpu()
    assert bool((got[:2] == 3).all()) and torch.equal(got[2:], want[2:])


@pytest.mark.parametrize("group", [32, 128])
def test_quantiser_at_the_borders(cuda, group):
    """Exact ties, constants, tiny and huge ranges, subnormals, a large offset, NaN and infinities."""
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(12, 1, 128)
    x[0, 0] = torch.arange(128) % 31 * 0.5            # range 15, scale 1: every half is a tie
    x[1] = 3.5
    x[2, 0] = torch.randn(128, generator=g) * 1e-38   # scale is subnormal
    x[3, 0] = torch.randn(128, generator=g) * 1e37
    x[4, 0] = 1000 + torch.arange(128) % 16 * 8.0
    x[5, 0] = torch.where(torch.arange(128) % 2 == 0, -7.5, 7.5)
    x[5, 0, 3::8] = torch.randn(16, generator=g) * 1e-9  # next to the tie in the middle
    x[6, 0, 7] = float("inf")
    x[7, 0, 99] = -float("inf")
    x[8, 0, 64] = float("nan")
    x[9, 0, :2] = torch.tensor([3.3e38, -3.3e38])     # the range is above the largest f32
    x[10, 0] = torch.randn(128, generator=g) * 2.0 ** -130
    x[11, 0] = -0.0
    x = x.to(torch.bfloat16)
    cache = make_cache([12], 1, group, cuda)
    cache.append(x.to(cuda), x.to(cuda))
    kf, vf = cache.read(12, dtype=torch.float32)
    want = kr.held(x, group)
    for got in (kf.cpu(), vf.cpu()):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.float().nan_to_num())


def test_many_random_groups_are_exact(cuda):
    """4 M values of several magnitudes: not one code differs from exact arithmetic."""
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(4096, 8, 128, generator=g, device=cuda)
    x = (x * torch.exp(6 * torch.randn(4096, 8, 1, generator=g, device=cuda))).to(torch.bfloat16)
    cache = make_cache([4096], 8, 32, cuda)
    cache.append(x, x)
    kf, vf = cache.read(4096, dtype=torch.float32)
    want = kr.held(x, 32).float()
    assert torch.equal(kf, want) and torch.equal(vf, want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

CASES = [
    # lens, rows a sequence, H, Hkv, group, causal
    ([1], 1, 1, 1, 128, True),
    ([77], 1, 32, 8, 128, True),
    ([64, 65, 63, 1, 129], 1, 8, 2, 32, True),
    ([300, 40, 1000], 1, 5, 5, 64, True),
    ([200, 77], 3, 14, 2, 32, True),      # 7 heads a K/V head, 21 rows
    ([90, 33, 50], 5, 8, 4, 64, True),
    ([90, 33, 50], 5, 8, 4, 64, False),
    ([70, 130], 2, 16, 1, 128, True),     # 32 rows of one K/V head
    ([500], 17, 3, 3, 32, True),
    ([33, 64, 100], 16, 16, 2, 128, False),
]


@pytest.mark.parametrize("lens,new,H,Hkv,group,causal", CASES)
def test_attention(cuda, lens, new, H, Hkv, group, causal):
    import ltxb
    cache, k, v = filled(lens, Hkv, group, cuda, seed=len(lens) + H)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(len(lens) * new, H, 128, generator=g).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache, causal=causal)
    torch.cuda.synchronize()
    assert ltxb.device_status() == ltxb.OK
    for b in range(len(lens)):
        want = kr.attention(q[b * new:(b + 1) * new], k[b], v[b], causal)
        check(out[b * new:(b + 1) * new], want, float(v[b].abs().max()), f"sequence {b}")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_ragged_rows_and_lengths(cuda, group, causal):
    """Sequences with no rows, no tokens, fewer tokens than rows; strided q; a gate; padding rows stay."""
    import ltxb
    lens, new, H, Hkv = [100, 0, 7, 300, 64, 3], [4, 2, 0, 1, 64, 5], 6, 3
    cache, k, v = filled(lens, Hkv, group, cuda, seed=4)
    rs = starts(new, cuda)
    n = sum(new)
    g = torch.Generator().manual_seed(10)
    fused = torch.randn(n + 3, 2 * H, 128, generator=g).to(torch.bfloat16).to(cuda)
    q = fused[:, H:]
    gate = torch.rand(n + 3, H, generator=g).to(cuda)
    out = torch.full((n + 3, H, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    ltxb.attention_kv4(q, cache, row_start=rs, causal=causal, gate=gate, scale=0.2, out=out)
    torch.cuda.synchronize()
    assert ltxb.device_status() == ltxb.OK
    at = 0
    for b, c in enumerate(new):
        want = kr.attention(q[at:at + c].cpu(), k[b], v[b], causal, scale=0.2, gate=gate[at:at + c])
        check(out[at:at + c], want, float(v[b].abs().max()) if lens[b] else 0.0, f"sequence {b}")
        at += c
    assert bool((out[n:] == 5).all())
    # the rows of the sequence without tokens, and those before a first token, are zeros and not small numbers
    assert bool((out[4:6] == 0).all())
    if causal:
        assert bool((out[n - 5:n - 3] == 0).all())


def test_attention_long_cache_many_pieces(cuda):
    """One sequence cut into a piece per CTA, and a batch where items end inside pieces; against f64 on the GPU."""
    import ltxb
    for lens, H, Hkv, group in (([40001], 4, 1, 128), ([5000, 1, 12345, 300], 16, 4, 32), ([33333], 2, 2, 64)):
        cache = make_cache(lens, Hkv, group, cuda, seed=7)
        k = rows_like((sum(lens), Hkv, 128), 1, cuda)
        v = rows_like((sum(lens), Hkv, 128), 2, cuda)
        cache.append(k, v, row_start=starts(lens, cuda))
        q = torch.randn(len(lens), H, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
        out = ltxb.attention_kv4(q, cache)
        kh, vh = kr.held(k, group).split(lens), kr.held(v, group).split(lens)
        for b in range(len(lens)):
            kk, vv = (t.repeat_interleave(H // Hkv, 1) for t in (kh[b], vh[b]))
            p = torch.softmax(torch.einsum("hd,thd->ht", q[b].double(), kk) / math.sqrt(128), -1)
            want = torch.einsum("ht,thd->hd", p, vv).cpu()
            check(out[b], want, float(vv.abs().max()), f"{lens} sequence {b}")
    assert ltxb.device_status() == ltxb.OK


def test_attention_peaked_and_growing_scores(cuda):
    """Scores that climb along the cache (the reference maximum and the V power move often), V of very unequal scale."""
    import ltxb
    T, H = 1500, 2
    k, v = rows_like((T, H, 128), 1, cuda).float(), rows_like((T, H, 128), 2, cuda).float()
    ramp = torch.linspace(0, 1, T, device=cuda)[:, None, None]
    q = torch.randn(1, H, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    k = (k + q.float() * ramp * 4).to(torch.bfloat16)
    v = (v * torch.exp2(20 * (ramp - 0.5))).to(torch.bfloat16)
    cache = make_cache([T], H, 64, cuda)
    cache.append(k, v)
    out = ltxb.attention_kv4(q, cache)
    kh, vh = kr.held(k, 64), kr.held(v, 64)
    p = torch.softmax(torch.einsum("hd,thd->ht", q[0].double(), kh) / math.sqrt(128), -1)
    want = torch.einsum("ht,thd->hd", p, vh)
    # the bound's |v| is that of the tokens that matter: the weighted mean of the row maxima
    vmax = (p[:, :, None] * vh.abs().amax(-1).T[:, :, None]).sum(1)
    err = (out[0].double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * vmax).all())


@pytest.mark.parametrize("causal", [True, False])
def test_nan_reaches_exactly_the_rows_that_see_it(cuda, causal):
    """A token with a NaN in its K or V: rows that attend to it are NaN, rows before it are not touched."""
    import ltxb
    T, H = 40, 2
    for which in ("k", "v"):
        k, v = rows_like((T, H, 128), 1, cuda), rows_like((T, H, 128), 2, cuda)
        (k if which == "k" else v)[30, 1, 17] = float("inf") if which == "k" else float("nan")
        cache = make_cache([T], H, 32, cuda)
        cache.append(k, v)
        q = torch.randn(T, H, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        out = ltxb.attention_kv4(q.to(cuda), cache, causal=causal).cpu()
        first = 30 if causal else 0
        assert bool(out[first:, 1].isnan().all())
        kh, vh = kr.held(k.cpu(), 32), kr.held(v.cpu(), 32)
        want = kr.attention(q[:, :1], kh[:, :1], vh[:, :1], causal)
        check(out[:, :1], want, float(vh[:, 0].abs().max()))
        if causal:
            want = kr.attention(q[:30, 1:], kh[:30, 1:], vh[:30, 1:], causal)
            check(out[:30, 1:], want, float(vh[:30, 1].abs().max()))


def test_shared_pages_and_order_of_pages(cuda):
    """Two sequences over the same first page (a shared prompt), the rest their own."""
    import ltxb
    cache, k, v = filled([100, 100], 2, 128, cuda, seed=3)
    cache.page_table[1, 0] = cache.page_table[0, 0]
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache)
    check(out[:1], kr.attention(q[:1], k[0], v[0], True), float(v[0].abs().max()))
    k1, v1 = torch.cat([k[0][:64], k[1][64:]]), torch.cat([v[0][:64], v[1][64:]])
    check(out[1:], kr.attention(q[1:], k1, v1, True), float(v1.abs().max()))


def test_no_page_table(cuda):
    import ltxb
    cache = ltxb.KV4Cache(batch=3, max_len=150, kv_heads=2, group=64, device=cuda)
    k, v = rows_like((3 * 150, 2, 128), 1, cuda), rows_like((3 * 150, 2, 128), 2, cuda)
    cache.seq_lens.fill_(150)
    cache.append(k, v)
    q = torch.randn(3, 2, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache)
    kh, vh = kr.held(k.cpu(), 64), kr.held(v.cpu(), 64)
    for b in range(3):
        s = slice(150 * b, 150 * b + 150)
        check(out[b:b + 1], kr.attention(q[b:b + 1], kh[s], vh[s], True), float(vh[s].abs().max()))


def test_bad_indexes_are_reported_and_not_followed(cuda):
    """A page number outside the pool, a length above the capacity, a row range outside the call."""
    import ltxb
    lens = [130, 70]
    q = torch.randn(2, 2, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    for bad in (-1, 1 << 30):
        cache, k, v = filled(lens, 2, 128, cuda, seed=3)
        cache.page_table[0, 1] = bad
        out = ltxb.attention_kv4(q.to(cuda), cache)
        rc, site = ltxb.device_status_site()
        assert rc == ltxb.EINVAL and site == ltxb.SITE_KV4_PAGE and "page" in ltxb.last_error()
        assert bool(out[0].isnan().all())
        check(out[1:], kr.attention(q[1:], k[1], v[1], True), float(v[1].abs().max()))
        kk = rows_like((200, 2, 128), 1, cuda)
        before = cache.pages.clone()
        cache.append(kk, kk, row_start=starts(lens, cuda))
        assert ltxb.device_status() == ltxb.EINVAL
        touched = {int(x) for x in (cache.pages != before).nonzero()[:, 0].unique()}
        assert touched <= {int(x) for x in cache.page_table.flatten().cpu() if 0 <= int(x) < cache.pages.shape[0]}
        o = tuple(torch.full((200, 2, 128), 9.0, device=cuda) for _ in range(2))
        cache.read(200, row_start=starts(lens, cuda), dtype=torch.float32, out=o)
        assert ltxb.device_status() == ltxb.EINVAL
        assert bool((o[0][64:128] == 9).all()) and not bool((o[0][:64] == 9).all())
    cache, k, v = filled(lens, 2, 128, cuda, seed=3)
    cache.seq_lens[1] = 1000  # capacity: 3 pages
    ltxb.attention_kv4(q.to(cuda), cache)
    rc, site = ltxb.device_status_site()
    assert rc == ltxb.EINVAL and site == ltxb.SITE_KV4_LEN
    cache.seq_lens[1] = -4
    out = ltxb.attention_kv4(q.to(cuda), cache)
    assert ltxb.device_status() == ltxb.EINVAL and bool((out[1] == 0).all())
    cache.seq_lens[1] = 70
    out = torch.full((2, 2, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    ltxb.attention_kv4(q.to(cuda), cache, row_start=torch.tensor([0, 1, 7], dtype=torch.int32, device=cuda), out=out)
    rc, site = ltxb.device_status_site()
    assert rc == ltxb.EINVAL and site == ltxb.SITE_KV4_ROWS
    assert ltxb.device_status() == ltxb.OK


def test_python_refusals(cuda):
    import ltxb
    cache = make_cache([10], 2, 64, cuda)
    k = rows_like((1, 2, 128), 1, cuda)
    for f in (lambda: cache.append(k.float(), k.float()), lambda: cache.append(k, k.repeat(2, 1, 1)),
              lambda: cache.append(k[:, :1], k[:, :1]), lambda: cache.append(k.cpu(), k.cpu()),
              lambda: cache.append(k.transpose(1, 2).contiguous().transpose(1, 2), k),
              lambda: cache.append(k, k, row_start=torch.zeros(3, dtype=torch.int32, device=cuda)),
              lambda: cache.append(k, k, row_start=torch.zeros(2, dtype=torch.int64, device=cuda)),
              lambda: cache.read(1, dtype=torch.float16), lambda: cache.read(1, out=(k, k[:0])),
              lambda: ltxb.attention_kv4(rows_like((1, 3, 128), 1, cuda), cache),
              lambda: ltxb.attention_kv4(k, cache, gate=torch.zeros(2, 2, device=cuda)),
              lambda: ltxb.attention_kv4(k, cache, out=k.float()),
              lambda: ltxb.attention_kv4(k, cache, workspace=torch.empty(256, dtype=torch.uint8, device=cuda)),
              lambda: ltxb.KV4Cache(1, 10, 1, group=16, device=cuda),
              lambda: ltxb.KV4Cache.from_pages(cache.pages, cache.page_table, cache.seq_lens, group=32),
              lambda: ltxb.KV4Cache.from_pages(cache.pages, cache.page_table.long(), cache.seq_lens, group=64)):
        with pytest.raises(ltxb.LtxbError):
            f()


def test_lengths_and_page_table_may_be_replaced(cuda):
    """A length or table tensor assigned to the cache is the one that is read."""
    import ltxb
    cache, k, v = filled([130, 40], 2, 64, cuda, seed=4)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    cache.seq_lens = cache.seq_lens - torch.tensor([70, 3], dtype=torch.int32, device=cuda)
    got = ltxb.attention_kv4(q, cache)
    for b, n in enumerate((60, 37)):
        check(got[b:b + 1], kr.attention(q[b:b + 1].cpu(), k[b][:n], v[b][:n], True), float(v[b].abs().max()))
    cache.page_table = cache.page_table.flip(0)  # the sequences change places
    cache.seq_lens = torch.tensor([40, 130], dtype=torch.int32, device=cuda)
    got = ltxb.attention_kv4(q, cache)
    for b in (0, 1):
        check(got[b:b + 1], kr.attention(q[b:b + 1].cpu(), k[1 - b], v[1 - b], True), float(v[1 - b].abs().max()))
    for bad in (None, cache.seq_lens.long(), cache.seq_lens[:1]):
        with pytest.raises(ltxb.LtxbError):
            cache.seq_lens = bad
    for bad in (None, cache.page_table[:1]):
        with pytest.raises(ltxb.LtxbError):
            cache.page_table = bad


def test_deterministic_and_on_another_stream(cuda):
    import ltxb
    cache, _, _ = filled([3000, 17, 900], 2, 32, cuda, seed=3)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    a = ltxb.attention_kv4(q, cache)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    b = ltxb.attention_kv4(q, cache, stream=st, out=torch.empty_like(q),
                           workspace=torch.empty(64 << 20, dtype=torch.uint8, device=cuda))
    st.synchronize()
    assert torch.equal(a, b)


def test_graph_replays_with_other_lengths_and_pages(cuda):
    """Decoding captured once: write a token, attend, with the lengths moving on between replays."""
    import ltxb
    H, Hkv, group = 8, 2, 64
    cache = make_cache([100, 60, 5], Hkv, group, cuda, max_pages=4)
    k0, v0 = rows_like((165, Hkv, 128), 1, cuda), rows_like((165, Hkv, 128), 2, cuda)
    cache.append(k0, v0, row_start=starts([100, 60, 5], cuda))
    hist = [[t] for t in k0.split([100, 60, 5])], [[t] for t in v0.split([100, 60, 5])]
    q, k, v = (torch.zeros(3, h, 128, dtype=torch.bfloat16, device=cuda) for h in (H, Hkv, Hkv))
    out = torch.empty_like(q)

    def step():
        cache.seq_lens.add_(1)
        cache.append(k, v)
        ltxb.attention_kv4(q, cache, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # first use outside the capture
        ltxb.attention_kv4(q, cache, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        q.copy_(torch.randn(3, H, 128, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        k.copy_(rows_like((3, Hkv, 128), 50 + i, cuda))
        v.copy_(rows_like((3, Hkv, 128), 80 + i, cuda))
        graph.replay()
        for b in range(3):
            hist[0][b].append(k[b:b + 1].clone())
            hist[1][b].append(v[b:b + 1].clone())
            kk, vv = (kr.held(torch.cat(t[b]).cpu(), group) for t in hist)
            check(out[b:b + 1], kr.attention(q[b:b + 1], kk, vv, True), float(vv.abs().max()), f"step {i}, {b}")
    assert ltxb.device_status() == ltxb.OK


# ---------------------------------------------------------------------------
# many rows: the tcgen05 kernel over f16 operands
# ---------------------------------------------------------------------------

def check_many(got, want, q, k, v, scale=None):
    """K and V are rounded to f16 (2^-11 each), P too, exp2 is off by at most
    2^-13: a score moves by at most 2^-11 scale sum |q_d k_d| =: 2^-11 A, so an
    output by 2^-10 A max|v| from the scores (numerator and denominator) and
    2^-9 max|v| from P, V and exp2, besides its own rounding. The roundings
    being independent, the 2-norm of the error stays near that of the output's
    rounding: bf16's root mean square error is at most 2^-8 / sqrt(3) = 2.3e-3
    of a value; 3e-3 leaves room for the others (2^-11 / sqrt(3) each)."""
    got = got.double().cpu()
    if got.numel() == 0:
        return
    scale = 1 / math.sqrt(128) if scale is None else scale
    a = scale * float((q.double().cpu().abs().amax((0, 1)) * k.abs().amax((0, 1))).sum())
    vmax = float(v.abs().max())
    err = (got - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + vmax * (2.0 ** -9 + 2.0 ** -10 * a)).all())
    n = float(want.norm())
    assert float((got - want).norm()) <= 3e-3 * n, float((got - want).norm()) / n


MANY = [
    # lens, rows a sequence, H, Hkv, group, causal
    ([64], 64, 1, 1, 128, True),
    ([300], 300, 2, 1, 32, True),
    ([257, 129], 128, 3, 3, 64, True),
    ([500, 100, 130], 100, 4, 2, 128, False),
    ([1000], 70, 7, 1, 32, True),          # 490 rows of one K/V head: a tile crosses tokens
    ([1500], 256, 1, 1, 64, False),        # one tile: the keys are split
    ([2000, 65], 65, 2, 2, 32, True),
]


@pytest.mark.parametrize("lens,new,H,Hkv,group,causal", MANY)
def test_many_rows(cuda, lens, new, H, Hkv, group, causal):
    import ltxb
    cache, k, v = filled(lens, Hkv, group, cuda, seed=len(lens) + H)
    q = torch.randn(len(lens) * new, H, 128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache, causal=causal)
    torch.cuda.synchronize()
    assert ltxb.device_status() == ltxb.OK
    for b in range(len(lens)):
        qb = q[b * new:(b + 1) * new]
        check_many(out[b * new:(b + 1) * new], kr.attention(qb, k[b], v[b], causal), qb, k[b], v[b])


@pytest.mark.parametrize("scale", [0.2, -0.1, 0.0])
@pytest.mark.parametrize("causal", [True, False])
def test_many_ragged_rows(cuda, causal, scale):
    """No rows, no tokens, fewer tokens than rows, one token; strided q, a gate, padding rows."""
    import ltxb
    lens, new, H, Hkv, group = [100, 0, 7, 300, 64, 3, 1, 513], [90, 20, 0, 300, 64, 50, 1, 200], 6, 2, 64
    cache, k, v = filled(lens, Hkv, group, cuda, seed=4)
    rs, n = starts(new, cuda), sum(new)
    g = torch.Generator().manual_seed(10)
    fused = torch.randn(n + 5, 2 * H, 128, generator=g).to(torch.bfloat16).to(cuda)
    q = fused[:, H:]
    gate = torch.rand(n + 5, H, generator=g).to(cuda)
    out = torch.full((n + 5, H, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    ltxb.attention_kv4(q, cache, row_start=rs, causal=causal, gate=gate, scale=scale, out=out)
    torch.cuda.synchronize()
    assert ltxb.device_status() == ltxb.OK
    at = 0
    for b, c in enumerate(new):
        if c:
            qb = q[at:at + c].cpu()
            want = kr.attention(qb, k[b], v[b], causal, scale=scale, gate=gate[at:at + c])
            if lens[b]:
                check_many(out[at:at + c], want, qb, k[b], v[b], scale=abs(scale))
            # rows that see nothing are zeros, whole (a single value of another row may come to 0 as well)
            assert torch.equal((out[at:at + c].cpu() == 0).all(-1), (want == 0).all(-1))
        at += c
    assert bool((out[n:] == 5).all())


def test_many_rows_over_long_keys_in_splits(cuda):
    import ltxb
    lens, new, H, Hkv, group = [9000, 3001], [200, 90], 4, 2, 128
    cache, k, v = filled(lens, Hkv, group, cuda, seed=1)
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    for causal in (True, False):
        out = ltxb.attention_kv4(q.to(cuda), cache, row_start=starts(new, cuda), causal=causal)
        again = ltxb.attention_kv4(q.to(cuda), cache, row_start=starts(new, cuda), causal=causal)
        assert torch.equal(out, again)
        at = 0
        for b, c in enumerate(new):
            pick = list(range(0, c, 17)) + [c - 1]
            for i in pick:
                seen = lens[b] - c + i + 1 if causal else lens[b]
                qi = q[at + i:at + i + 1]
                want = kr.attention(qi, k[b][:seen], v[b][:seen], False)
                check_many(out[at + i:at + i + 1], want, qi, k[b], v[b])
            at += c
    assert ltxb.device_status() == ltxb.OK


@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_nan_and_bad_pages(cuda, causal):
    import ltxb
    T, H = 300, 2
    q = torch.randn(T, H, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    for which in ("k", "v", "page"):
        k, v = rows_like((T, H, 128), 1, cuda), rows_like((T, H, 128), 2, cuda)
        if which != "page":
            (k if which == "k" else v)[130, 1, 17] = float("nan")
        cache = make_cache([T], H, 32, cuda)
        cache.append(k, v)
        if which == "page":
            cache.page_table[0, 2] = 1 << 20
        out = ltxb.attention_kv4(q.to(cuda), cache, causal=causal).cpu()
        assert ltxb.device_status() == (ltxb.EINVAL if which == "page" else ltxb.OK)
        first = (128 if which == "page" else 130) if causal else 0
        assert bool(out[first:, 1].isnan().all())
        kh, vh = kr.held(k.cpu(), 32), kr.held(v.cpu(), 32)
        heads = [0] if which != "page" else []
        for h in heads:
            check_many(out[:, h:h + 1], kr.attention(q[:, h:h + 1], kh[:, h:h + 1], vh[:, h:h + 1], causal),
                       q[:, h:h + 1], kh[:, h:h + 1], vh[:, h:h + 1])
        if causal:
            check_many(out[:first, 1:], kr.attention(q[:first, 1:], kh[:first, 1:], vh[:first, 1:], True),
                       q[:first, 1:], kh[:first, 1:], vh[:first, 1:])


def test_many_rows_of_unequal_size(cuda):
    """Rows, keys and values over many powers of two: the f16 operands' powers take them in."""
    import ltxb
    T, H = 200, 2
    g = torch.Generator().manual_seed(3)
    for qs, ks, vs in ((1e-30, 1e30, 1e-30), (1e25, 1e-25, 1e30), (1.0, 1.0, 1e-37), (1e-38, 1e-5, 1.0)):
        q = (torch.randn(T, H, 128, generator=g) * qs * torch.exp2(torch.arange(T) % 5 - 2.0)[:, None, None]).to(torch.bfloat16)
        k, v = (torch.randn(T, H, 128, generator=g) * s for s in (ks, vs))
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        cache = make_cache([T], H, 64, cuda)
        cache.append(k.to(cuda), v.to(cuda))
        out = ltxb.attention_kv4(q.to(cuda), cache)
        kh, vh = kr.held(k, 64), kr.held(v, 64)
        check_many(out, kr.attention(q, kh, vh, True), q, kh, vh)


def test_capacity_far_above_the_lengths(cuda):
    """A page table with room for 200 pages a sequence and a bound known on the host; lengths replayed in a graph."""
    import ltxb
    H, Hkv, group, new = 4, 2, 32, 48
    cache = make_cache([100, 60], Hkv, group, cuda, max_pages=200)
    bound = ltxb.KV4Cache.from_pages(cache.pages, cache.page_table, cache.seq_lens, group=group, max_len=700)
    k, v = rows_like((1400, Hkv, 128), 1, cuda), rows_like((1400, Hkv, 128), 2, cuda)
    cache.seq_lens.fill_(700)
    cache.append(k, v)
    kh, vh = kr.held(k.cpu(), group).view(2, 700, Hkv, 128), kr.held(v.cpu(), group).view(2, 700, Hkv, 128)
    q = torch.randn(2 * new, H, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    out = torch.empty_like(q)
    ltxb.attention_kv4(q, bound, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ltxb.attention_kv4(q, bound, out=out)
    for lens in ([700, 699], [100, 48], [64, 640]):
        cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        for b, n in enumerate(lens):
            qb = q[b * new:(b + 1) * new].cpu()
            check_many(out[b * new:(b + 1) * new], kr.attention(qb, kh[b, :n], vh[b, :n], True), qb, kh[b, :n], vh[b, :n])
    assert ltxb.device_status() == ltxb.OK
    cache.seq_lens.fill_(701)
    ltxb.attention_kv4(q, bound, out=out)
    assert ltxb.device_status_site() == (ltxb.EINVAL, ltxb.SITE_KV4_LEN)


# ---------------------------------------------------------------------------
# as they are used together, and at the edges
# ---------------------------------------------------------------------------

def test_a_decoder_layer_step_by_step(cuda):
    """Prompt rows and then single tokens through 4-bit projections, the cache
    and the attention, against the same steps in f64 on what each holds (the
    projections' outputs are rounded to bf16 as the operators round them)."""
    import ltxb
    D, H, Hkv, group, B = 512, 4, 2, 64, 3
    lens = [70, 5, 130]
    g = torch.Generator(device=cuda).manual_seed(0)
    wq = [ltxb.quantize_g4(torch.randn(n, D, generator=g, device=cuda) / D ** 0.5, group)
          for n in ((H + 2 * Hkv) * 128, D)]
    full = []
    for c, s in wq:
        code = torch.stack((c & 15, c >> 4), -1).flatten(-2).double() - 8
        full.append(code * s.double().repeat_interleave(group, 1))
    cache = make_cache(lens, Hkv, group, cuda, max_pages=4)
    cache.seq_lens.zero_()
    hist = [[], []]

    def layer(x, counts):
        n = x.shape[0]
        cache.seq_lens.add_(torch.tensor(counts, dtype=torch.int32, device=cuda))
        rs = starts(counts, cuda)
        qkv = ltxb.dq4_gemm(x, *wq[0]).view(n, H + 2 * Hkv, 128)
        q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        cache.append(k, v, row_start=rs)
        o = ltxb.attention_kv4(q, cache, row_start=rs)
        y = ltxb.dq4_gemm(o.view(n, H * 128), *wq[1])
        # the same in f64 from the operators' own bf16 intermediates, one step at a time
        want = x.double() @ full[0].T
        err = (qkv.view(n, -1).double() - want).abs()
        # M > 64 rounds the weights to bf16 first: six root mean squares of 2^-8
        norm = (x.double() ** 2 @ full[0].T ** 2).sqrt()
        assert bool((err <= 2.0 ** -8 * want.abs() + 6 * 2.0 ** -8 * norm).all())
        at = 0
        for b, c in enumerate(counts):
            hist[0].append((b, k[at:at + c].clone()))
            hist[1].append((b, v[at:at + c].clone()))
            kk, vv = (kr.held(torch.cat([t for i, t in h if i == b]).cpu(), group) for h in hist)
            w = kr.attention(q[at:at + c].cpu(), kk, vv, True)
            check_many(o[at:at + c], w, q[at:at + c].cpu(), kk, vv)
            at += c
        want = o.view(n, -1).double() @ full[1].T
        norm = (o.view(n, -1).double() ** 2 @ full[1].T ** 2).sqrt()
        assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 6 * 2.0 ** -8 * norm).all())
        return y
    x = torch.randn(sum(lens), D, generator=g, device=cuda).to(torch.bfloat16)
    layer(x, lens)
    for step in range(3):
        layer(torch.randn(B, D, generator=g, device=cuda).to(torch.bfloat16), [1] * B)
    assert ltxb.device_status() == ltxb.OK


def test_many_sequences(cuda):
    """More sequences than a CTA has threads, empty ones among them; uniform and ragged rows."""
    import ltxb
    B, H, Hkv, group = 300, 4, 2, 32
    lens = [(37 * b) % 200 for b in range(B)]
    cache, k, v = filled(lens, Hkv, group, cuda, seed=2)
    q = torch.randn(B, H, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache)
    again = ltxb.attention_kv4(q.to(cuda), cache, row_start=starts([1] * B, cuda))
    assert torch.equal(out, again)
    for b in list(range(0, B, 23)) + [B - 1]:
        want = kr.attention(q[b:b + 1], k[b], v[b], True)
        check(out[b:b + 1], want, float(v[b].abs().max()) if lens[b] else 0.0, f"sequence {b}")
    assert bool((out[[b for b in range(B) if lens[b] == 0]] == 0).all())
    assert ltxb.device_status() == ltxb.OK


def test_offsets_beyond_32_bits(cuda):
    """A pool of more than 4 GB whose last pages are used."""
    import ltxb
    block = ltxb.lib.ltxb_kv4_block_bytes(128)
    n = (1 << 32) // (block * 8) + 40
    pages = torch.empty(n, 8, block, dtype=torch.uint8, device=cuda)
    lens = [200, 90]
    table = torch.tensor([[n - 1, 3, n - 2, n - 5], [n - 7, n - 3, 0, 1]], dtype=torch.int32, device=cuda)
    cache = ltxb.KV4Cache.from_pages(pages, table, torch.tensor(lens, dtype=torch.int32, device=cuda), group=128)
    k, v = rows_like((290, 8, 128), 1, cuda), rows_like((290, 8, 128), 2, cuda)
    rs = starts(lens, cuda)
    cache.append(k, v, row_start=rs)
    kh, vh = kr.held(k.cpu(), 128), kr.held(v.cpu(), 128)
    kf, vf = cache.read(290, row_start=rs, dtype=torch.float32)
    assert torch.equal(kf.cpu(), kh.float()) and torch.equal(vf.cpu(), vh.float())
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = ltxb.attention_kv4(q.to(cuda), cache)
    many = torch.randn(180, 8, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out2 = ltxb.attention_kv4(many.to(cuda), cache)
    for b, at in ((0, 0), (1, 200)):
        kk, vv = kh[at:at + lens[b]], vh[at:at + lens[b]]
        check(out[b:b + 1], kr.attention(q[b:b + 1], kk, vv, True), float(vv.abs().max()))
        qb = many[90 * b:90 * b + 90]
        check_many(out2[90 * b:90 * b + 90], kr.attention(qb, kk, vv, True), qb, kk, vv)


def test_two_streams_at_once(cuda):
    """Calls over two caches on two streams, each with the workspace of its own call."""
    import ltxb
    caches = [filled([2000, 700], 4, g, cuda, seed=i) for i, g in enumerate((32, 128))]
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    many = torch.randn(2 * 96, 8, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    alone = [[ltxb.attention_kv4(x, c[0]) for x in (q, many)] for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(4):
        for i, (c, st) in enumerate(zip(caches, streams)):
            with torch.cuda.stream(st):
                got[i].append([ltxb.attention_kv4(x, c[0]) for x in (q, many)])
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(pair, alone[i]))
    # a stream given by name, not the current one
    a = ltxb.attention_kv4(q, caches[0][0], stream=streams[1])
    streams[1].synchronize()
    assert torch.equal(a, alone[0][0])


def test_infinite_and_nan_queries_stay_in_their_rows(cuda):
    import ltxb
    cache, k, v = filled([150], 2, 64, cuda, seed=2)
    for n in (6, 100):
        q = torch.randn(n, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        clean = ltxb.attention_kv4(q.to(cuda), cache)
        bad = q.clone()
        bad[2, 1, 5] = float("nan")
        bad[3, 0, 7] = float("inf")
        out = ltxb.attention_kv4(bad.to(cuda), cache)
        assert bool(out[2, 1].isnan().all()) and bool(out[3, 0].isnan().all())
        keep = torch.ones(n, 4, dtype=torch.bool)
        keep[2, 1] = keep[3, 0] = False
        assert torch.equal(out[keep.to(cuda)], clean[keep.to(cuda)])


def test_sequences_without_rows_are_left_alone(cuda):
    """An idle slot of a batch (no rows in the call, a length, page numbers that
    mean nothing) is neither read nor reported, nor are rows behind the last."""
    import ltxb
    cache, k, v = filled([100, 61, 5], 2, 64, cuda, seed=6)
    table = cache.page_table.clone()
    table[1:] = 1 << 29
    cache.page_table = table
    before = cache.pages.clone()
    for n in (2, 100):  # the last rows of the first sequence; the page kernel and the tcgen05 one
        rs = starts([n, 0, 0], cuda)
        kk, vv = cache.read(n, row_start=rs, dtype=torch.float32)
        assert torch.equal(kk.cpu().double(), k[0][100 - n:]) and torch.equal(vv.cpu().double(), v[0][100 - n:])
        q = torch.randn(n, 160, 128, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(cuda)
        want = kr.attention(q.cpu(), k[0], v[0], True)
        got = ltxb.attention_kv4(q[:, :160], cache, row_start=rs)
        if n == 2:
            check(got, want, float(v[0].abs().max()))
        else:
            check_many(got, want, q, k[0], v[0])
    # written again from where it was read: the same bytes, and nothing else's
    kb, vb = cache.read(3, row_start=starts([3, 0, 0], cuda))
    cache.seq_lens = torch.tensor([0, 61, 5], dtype=torch.int32, device=cuda)
    cache.append(kb[:0], vb[:0], row_start=starts([0, 0, 0], cuda))
    cache.append(kb, vb, row_start=starts([0, 0, 0], cuda))
    assert torch.equal(cache.pages, before)
    assert ltxb.device_status() == ltxb.OK


def test_infinite_queries_in_split_keys(cuda):
    """A row whose every score is minus infinity is NaN too, in one piece and in several."""
    import ltxb
    k, v = rows_like((1500, 1, 128), 1, cuda), rows_like((1500, 1, 128), 2, cuda)
    k[:, :, 7] = -50.0
    cache = make_cache([1500], 1, 32, cuda)
    cache.append(k, v)
    for n in (3, 256):
        q = torch.randn(n, 1, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
        clean = ltxb.attention_kv4(q, cache, causal=False)
        q[1, 0, 7] = float("inf")
        out = ltxb.attention_kv4(q, cache, causal=False)
        assert bool(out[1].isnan().all())
        keep = [i for i in range(n) if i != 1]
        assert torch.equal(out[keep], clean[keep])
