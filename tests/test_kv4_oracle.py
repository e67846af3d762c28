"""CPU tests of the 4-bit cache's oracle and of the entry points' refusals
(everything the host checks is refused before any device call)."""

import ctypes

import pytest
import torch

from oracle import kv4_ref as kr


def test_bf16_rounding_matches_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4096, generator=g) * torch.exp(8 * torch.randn(4096, generator=g))
    assert torch.equal(kr.bf16(x.double()), x.to(torch.bfloat16).double())


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantiser_error_is_half_a_step(group):
    """|x - held| <= scale / 2, plus what rounding the scale to bf16 (half a
    step, 2^-8 relative) takes off the top code's reach: 15 * 2^-8 scale."""
    g = torch.Generator().manual_seed(group)
    x = (torch.randn(50, 128, generator=g) * 3 + 1).to(torch.bfloat16)
    code, scale, zero = kr.quantise(x, group)
    err = (kr.values(code, scale, zero) - x.double()).abs()
    assert bool((err <= scale.repeat_interleave(group, -1) * (0.5 + 15 * 2.0 ** -8)).all())
    assert int(code.min()) >= 0 and int(code.max()) <= 15


def test_quantiser_edges():
    x = torch.zeros(4, 128)
    x[1] = 7.25                       # a constant group
    x[2, 5] = float("inf")
    x[3, 100] = float("nan")
    h = kr.held(x.to(torch.bfloat16), 32)
    assert torch.equal(h[0], torch.zeros(128).double())
    assert torch.equal(h[1], torch.full((128,), 7.25).double())
    assert bool(h[2, :32].isnan().all()) and torch.equal(h[2, 32:], torch.zeros(96).double())
    assert bool(h[3, 96:].isnan().all()) and torch.equal(h[3, :96], torch.zeros(96).double())


def _cache(ltxb, **kw):
    buf = ctypes.create_string_buffer(1 << 16)
    at = (ctypes.addressof(buf) + 255) & ~255
    f = dict(pages=at, page_table=at, seq_lens=at, n_pages=4, kv_heads=2, group=128, batch=2, max_pages=2, max_len=0)
    f.update(kw)
    c = ltxb._KV4(f["pages"], f["page_table"], f["seq_lens"], f["n_pages"], f["kv_heads"], f["group"], f["batch"],
                  f["max_pages"], f["max_len"])
    c._keep = buf
    return c, at


BAD_CACHES = [
    (dict(group=48), "group"), (dict(group=0), "group"), (dict(kv_heads=0), "heads"), (dict(n_pages=0), "pages"),
    (dict(batch=-1), "negative"), (dict(max_pages=-1), "negative"), (dict(max_len=-5), "negative"),
    (dict(pages=None), "missing"), (dict(seq_lens=None), "missing"), (dict(page_table=None, n_pages=3), "page table"),
    (dict(max_pages=1 << 26), "2\\^31"), (dict(batch=0), "no sequences"),
]


@pytest.mark.parametrize("bad,word", BAD_CACHES)
def test_bad_caches_are_refused(bad, word):
    import ltxb
    c, at = _cache(ltxb, **bad)
    r = ctypes.byref(c)
    n0 = ltxb.launch_count()
    for rc in (ltxb.lib.ltxb_kv4_append(r, None, at, 256, at, 256, 4, None),
               ltxb.lib.ltxb_kv4_read(r, None, at, at, ltxb.DT_BF16, 4, None),
               ltxb.lib.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, 0.1, at, 1 << 40, None)):
        assert rc == ltxb.EINVAL
        import re
        assert re.search(word, ltxb.last_error()), ltxb.last_error()
    assert ltxb.launch_count() == n0


def test_bad_arguments_are_refused():
    import ltxb
    c, at = _cache(ltxb)
    r = ctypes.byref(c)
    L, big = ltxb.lib, 1 << 40
    n0 = ltxb.launch_count()
    refused = [
        L.ltxb_kv4_append(None, None, at, 256, at, 256, 4, None),
        L.ltxb_kv4_append(r, None, at, 256, at, 256, 3, None),          # 3 rows, 2 sequences
        L.ltxb_kv4_append(r, None, at, 256, at, 256, -2, None),
        L.ltxb_kv4_append(r, None, at + 2, 256, at, 256, 4, None),      # misaligned
        L.ltxb_kv4_append(r, None, at, 252, at, 256, 4, None),          # stride not a multiple of 8
        L.ltxb_kv4_append(r, None, at, 256, at, 248, 4, None),          # stride below kv_heads * 128
        L.ltxb_kv4_append(r, None, None, 256, at, 256, 4, None),
        L.ltxb_kv4_append(r, at + 2, at, 256, at, 256, 4, None),        # row_start misaligned
        L.ltxb_kv4_read(r, None, at, at, ltxb.DT_I8, 4, None),
        L.ltxb_kv4_read(r, None, at, at + 8, ltxb.DT_F32, 4, None),
        L.ltxb_kv4_read(r, None, None, at, ltxb.DT_F32, 4, None),
        L.ltxb_attention_kv4(r, None, at, 384, at, None, 4, 3, 1, 0.1, at, big, None),   # 3 heads over 2
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 0, 1, 0.1, at, big, None),
        L.ltxb_attention_kv4(r, None, at, 128, at, None, 4, 2, 1, 0.1, at, big, None),   # stride below H * 128
        L.ltxb_attention_kv4(r, None, at + 8, 256, at, None, 4, 2, 1, 0.1, at, big, None),
        L.ltxb_attention_kv4(r, None, at, 256, at, at + 1, 4, 2, 1, 0.1, at, big, None),  # gate misaligned
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, float("nan"), at, big, None),
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, float("inf"), at, big, None),
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, 0.1, at, 64, None),    # small workspace
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, 0.1, at + 64, big, None),
        L.ltxb_attention_kv4(r, None, at, 256, at, None, 4, 2, 1, 0.1, None, big, None),
    ]
    assert refused == [ltxb.EINVAL] * len(refused)
    assert ltxb.launch_count() == n0
    assert L.ltxb_kv4_block_bytes(32) == 10240 and L.ltxb_kv4_block_bytes(64) == 9216
    assert L.ltxb_kv4_block_bytes(128) == 8704 and L.ltxb_kv4_block_bytes(16) == 0
    assert L.ltxb_attention_kv4_workspace_bytes(r, 4, 3) == 0 and L.ltxb_attention_kv4_workspace_bytes(r, 4, 4) > 0


def test_no_rows_is_no_work():
    import ltxb
    c, at = _cache(ltxb, batch=0)
    r = ctypes.byref(c)
    n0 = ltxb.launch_count()
    assert ltxb.lib.ltxb_kv4_append(r, None, None, 256, None, 256, 0, None) == ltxb.OK
    assert ltxb.lib.ltxb_kv4_read(r, None, None, None, ltxb.DT_BF16, 0, None) == ltxb.OK
    assert ltxb.lib.ltxb_attention_kv4(r, None, None, 256, None, None, 0, 2, 1, 0.1, None, 0, None) == ltxb.OK
    assert ltxb.launch_count() == n0


def test_bad_4bit_linear_calls_are_refused():
    import ltxb
    buf = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buf) + 255) & ~255
    f, big = ltxb.lib.ltxb_dq4_gemm, 1 << 40
    n0 = ltxb.launch_count()

    def call(A=at, W=at, S=at, dt=ltxb.DT_F32, group=128, bias=None, out=at, M=1, N=32, K=128, ws=at, wb=big):
        return f(A, W, S, dt, group, bias, out, M, N, K, ws, wb, None)
    refused = [call(dt=ltxb.DT_I8), call(group=16), call(group=256), call(M=-1), call(N=0), call(N=48), call(K=64),
               call(K=0), call(A=at + 2), call(A=None), call(W=at + 8), call(W=None), call(S=at + 4), call(S=None),
               call(out=at + 2), call(out=None), call(bias=at + 2), call(M=1025, wb=100), call(M=1025, ws=None),
               call(M=1025, ws=at + 8), call(M=9, ws=None), call(M=9, wb=100), call(M=9, ws=at + 8)]
    assert refused == [ltxb.EINVAL] * len(refused)
    assert call(M=0, A=None, W=None) == ltxb.OK
    assert ltxb.launch_count() == n0
    assert ltxb.lib.ltxb_dq4_gemm_workspace_bytes(1, 32, 128) == 0
    assert ltxb.lib.ltxb_dq4_gemm_workspace_bytes(1025, 32, 128) == 32 * 128 * 2
    assert ltxb.lib.ltxb_dq4_gemm_workspace_bytes(1024, 32, 128) == 0
