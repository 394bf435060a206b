"""Refusals of the attention operators and of the paged cache, checked before anything reaches a GPU."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

P = 1 << 20  # a 16-byte aligned address that is never followed


@pytest.fixture(scope="module")
def L():
    from miroxen_b200 import _lib, build
    if not _lib.lib_path().exists():
        build.build()
    return _lib


def cache(L, **more):
    c = L.KvCacheArgs(P, P, P, None, None, 10, 16 * 8 * 128, 8 * 128, 128, 4, 3, 4, 16, 8, 128, 0)
    for k, v in more.items():
        setattr(c, k, v)
    return c


def append(L, **more):
    a = L.AppendArgs(P, P, P, 3, 32 * 128, 8 * 128, 8 * 128, P, P, P, P, 64, P, P, None, P, None, 32, 128, 2, 1e-6)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def decode(L, **more):
    a = L.DecodeArgs(P, 32 * 128, P, P, P, P, 1 << 40, -1, 0, 32, 0.1)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def window(L, **more):
    a = L.AttnArgs(P, P, P, P, P, P, P, 100, 100, 32 * 128, 8 * 128, 8 * 128, 32 * 128, -1, 0, 0, 2, 32, 8, 128, 0.1)
    for k, v in more.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [dict(type=2), dict(D=0), dict(D=132), dict(D=136), dict(D=-8), dict(type=1, D=72), dict(Hkv=0), dict(page_size=0),
             dict(n_seqs=-1), dict(max_pages=-1), dict(num_pages=-1), dict(page_stride=4), dict(token_stride=1027), dict(head_stride=-128),
             dict(head_stride=64), dict(token_stride=0), dict(k=P + 8), dict(v=P + 2), dict(k_scale=P), dict(v_scale=P),
             dict(type=1, token_stride=1032)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches_are_refused_everywhere(L, bad):
    lib = L.lib()
    c = cache(L, **bad)
    assert lib.mxk_qkv_norm_rope_append(append(L), c, None) == -1
    assert b"qkv_norm_rope_append" in lib.mxk_last_error()
    if bad != dict(n_seqs=-1):
        assert lib.mxk_attn_decode_paged(decode(L), c, None) == -1
        assert b"attn_decode_paged" in lib.mxk_last_error()
    assert lib.mxk_attn_decode_workspace_bytes(c, 32) == -1


def test_too_many_tokens_per_sequence(L):
    lib = L.lib()
    c = cache(L, max_pages=1 << 27)
    assert lib.mxk_qkv_norm_rope_append(append(L), c, None) == -3
    assert lib.mxk_attn_decode_paged(decode(L), c, None) == -3
    c = cache(L, n_seqs=1 << 20, max_pages=1 << 20)
    assert lib.mxk_attn_decode_paged(decode(L), c, None) == -3


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(positions=None), dict(q=P + 2),
                                 dict(k=P + 8), dict(v=P + 4), dict(q_out=P + 8), dict(k_out=P + 8), dict(q_stride=4097), dict(k_stride=-8),
                                 dict(H=0), dict(H=-4), dict(mode=3), dict(rot=130), dict(rot=3), dict(rot=-2), dict(cos=None),
                                 dict(sin=None)], ids=str)
def test_append_refusals(L, bad):
    lib = L.lib()
    assert lib.mxk_qkv_norm_rope_append(append(L, **bad), cache(L), None) == -1
    assert b"qkv_norm_rope_append" in lib.mxk_last_error()


def test_append_null_structs_and_noops(L):
    lib = L.lib()
    assert lib.mxk_qkv_norm_rope_append(None, cache(L), None) == -1
    assert lib.mxk_qkv_norm_rope_append(append(L), None, None) == -1
    assert lib.mxk_qkv_norm_rope_append(append(L), cache(L, k=None), None) == -1
    assert lib.mxk_qkv_norm_rope_append(append(L), cache(L, page_table=None), None) == -1
    assert lib.mxk_qkv_norm_rope_append(append(L, T=1 << 31), cache(L), None) == -3
    assert lib.mxk_qkv_norm_rope_append(append(L, T=0), None, None) == 0
    assert lib.mxk_qkv_norm_rope_append(append(L, T=-2, q=None), cache(L), None) == 0


@pytest.mark.parametrize("D", [72, 128])
def test_append_refuses_more_heads_than_it_can_count(L, D):
    """In a process of its own: such a call has ended in a division by zero."""
    code = f"""import sys; sys.path.insert(0, {str(Path(__file__).parent)!r}); sys.path.insert(0, {str(Path(__file__).parent.parent)!r})
import test_cpu_attention as t
from miroxen_b200 import _lib as L
for H, Hkv in ((2**31 - 1, 2**30), (2**31 - 1, 1), (8, 2**31 - 1), (2**30 - 2, 1)):
    assert L.lib().mxk_qkv_norm_rope_append(t.append(L, H=H, rot={D}, q_stride=0), t.cache(L, Hkv=Hkv, D={D}, head_stride={D}), None) == -3, (H, Hkv)
    assert b"qkv_norm_rope_append" in L.lib().mxk_last_error()
"""
    subprocess.run([sys.executable, "-c", code], check=True)


@pytest.mark.parametrize("bad", [dict(q=None), dict(seq_lens=None), dict(out=None), dict(workspace=None), dict(q=P + 2), dict(out=P + 8),
                                 dict(workspace=P + 4), dict(workspace_bytes=4096), dict(workspace_bytes=-1), dict(q_stride=12), dict(q_stride=-8), dict(sinks=-1), dict(scale=0.0),
                                 dict(scale=-1.0), dict(scale=2e30), dict(scale=float("nan")), dict(scale=float("inf")), dict(H=0), dict(H=12)], ids=str)
def test_decode_refusals(L, bad):
    lib = L.lib()
    assert lib.mxk_attn_decode_paged(decode(L, **bad), cache(L), None) == -1
    assert b"attn_decode_paged" in lib.mxk_last_error()


def test_decode_null_structs_and_noops(L):
    lib = L.lib()
    assert lib.mxk_attn_decode_paged(None, cache(L), None) == -1
    assert lib.mxk_attn_decode_paged(decode(L), None, None) == -1
    assert lib.mxk_attn_decode_paged(decode(L), cache(L, v=None), None) == -1
    assert lib.mxk_attn_decode_paged(decode(L, q=None), cache(L, n_seqs=0), None) == 0
    assert lib.mxk_attn_decode_workspace_bytes(cache(L), 12) == -1


def test_decode_needs_a_page_table_wherever_it_may_look_into_it(L):
    lib = L.lib()
    for more in (dict(), dict(num_pages=0), dict(num_pages=0, k=None, v=None), dict(num_pages=0, type=1)):
        assert lib.mxk_attn_decode_paged(decode(L), cache(L, page_table=None, **more), None) == -1
        assert b"attn_decode_paged" in lib.mxk_last_error() and b"page table" in lib.mxk_last_error()


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=P + 2), dict(k=P + 8), dict(v=P + 4),
                                 dict(out=P + 8), dict(k_rows=-1), dict(H=0), dict(Hkv=0), dict(H=12), dict(D=4), dict(D=130), dict(D=136),
                                 dict(cu_q=None), dict(cu_k=None), dict(cu_q=None, cu_k=None), dict(q_stride=4092), dict(q_stride=4088),
                                 dict(k_stride=1016), dict(v_stride=0), dict(out_stride=-4096), dict(sinks=-1), dict(scale=0.0),
                                 dict(scale=float("nan")), dict(scale=float("inf"))], ids=str)
def test_window_refusals(L, bad):
    lib = L.lib()
    assert lib.mxk_attn_window(window(L, **bad), None) == -1
    assert b"attn_window" in lib.mxk_last_error()


def test_window_sizes_and_noops(L):
    lib = L.lib()
    assert lib.mxk_attn_window(None, None) == -1
    assert lib.mxk_attn_window(window(L, q_rows=1 << 30), None) == -3
    assert lib.mxk_attn_window(window(L, k_rows=1 << 31), None) == -3
    assert lib.mxk_attn_window(window(L, q_rows=0, q=None), None) == 0
    assert lib.mxk_attn_window(window(L, q_rows=-5), None) == 0
    assert lib.mxk_attn_window(window(L, n_seqs=0), None) == 0


def test_struct_sizes_match_the_header(L):
    assert C.sizeof(L.KvCacheArgs) == 5 * 8 + 5 * 8 + 6 * 4
    assert C.sizeof(L.AppendArgs) == 3 * 8 + 4 * 8 + 4 * 8 + 8 + 5 * 8 + 4 * 4
    assert C.sizeof(L.DecodeArgs) == 6 * 8 + 3 * 8 + 2 * 4
    assert C.sizeof(L.AttnArgs) == 7 * 8 + 9 * 8 + 4 * 4 + 8


def test_cache_handle_checks_its_tensors(L):
    import miroxen_b200 as mx
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 3, dtype=torch.int32)
    c = mx.KvCache(k, k.clone(), table)
    assert (c._args.num_pages, c._args.page_size, c._args.Hkv, c._args.D, c._args.type) == (4, 16, 2, 64, 0)
    assert (c._args.page_stride, c._args.token_stride, c._args.head_stride) == (2048, 128, 64)
    heads_first = torch.zeros(4, 2, 16, 64, dtype=torch.float8_e4m3fn)
    c = mx.KvCache(heads_first.transpose(1, 2), heads_first.clone().transpose(1, 2), table, torch.ones(2), torch.ones(2))
    assert (c._args.token_stride, c._args.head_stride, c._args.type) == (64, 1024, 1)
    for bad in [(k.float(), k.float(), table), (k, k[:3], table), (k, k.transpose(1, 2).contiguous().transpose(1, 2), table),
                (k.transpose(2, 3), k.transpose(2, 3), table), (k, k, table.long()), (k, k, table[0]), (k, k, table.t()),
                (k, k, table, torch.ones(2)), (heads_first, heads_first, table, torch.ones(3)),
                (heads_first, heads_first, table, torch.ones(16).double())]:
        with pytest.raises(mx.MxkError):
            mx.KvCache(*bad)
    with pytest.raises(mx.MxkError):
        mx.qkv_norm_rope_append(P, P, P, 1, 2, 128, None, None, 1e-6, None, None, 0, 0, 0, mx.KvCache(k, k.clone(), table), P, P)


def test_tensors_of_another_type_or_place_never_reach_the_library(L, monkeypatch):
    """Every tensor of each call in turn on the host, or of another type: refused by name, before its address goes anywhere."""
    import miroxen_b200 as mx
    from miroxen_b200 import ops

    class Reached:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    class OnGpu(torch.Tensor):  # says that it is on the current device
        def get_device(self):
            return 0

    def on(t):
        return t.as_subclass(OnGpu)

    monkeypatch.setattr(ops, "lib", lambda: Reached())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda i: 0)
    bf = torch.zeros(4, 256, dtype=torch.bfloat16)
    f, i = torch.zeros(4, 64), torch.zeros(5, dtype=torch.int32)
    pages, table = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 3, dtype=torch.int32)
    cache = mx.KvCache(pages, pages, table)
    cache._index = 0
    calls = {
        "qkv_norm_rope_append": (lambda a: mx.qkv_norm_rope_append(a["q"], a["k"], a["v"], 4, 4, 64, a["qw"], a["kw"], 1e-6, a["cos"], a["sin"], 4, 64, 2, cache,
                                                                   a["pos"], a["q_out"], seq_ids=a["ids"], rope_rows=a["rows"], k_out=a["k_out"]),
                                 dict(q=bf, k=bf, v=bf, qw=f, kw=f, cos=f, sin=f, pos=i, q_out=bf, ids=i, rows=i, k_out=bf)),
        "attn_decode_paged": (lambda a: mx.attn_decode_paged(a["q"], cache, a["lens"], 4, 0.1, a["out"], lse=a["lse"], workspace=a["ws"]),
                              dict(q=bf, lens=i, out=bf, lse=f, ws=torch.zeros(64, dtype=torch.uint8))),
        "attn_window": (lambda a: mx.attn_window(a["q"], a["k"], a["v"], 4, 4, 4, 4, 64, 0.1, a["out"], cu_q=a["cu_q"], cu_k=a["cu_k"], lse=a["lse"]),
                        dict(q=bf, k=bf, v=bf, out=bf, cu_q=i, cu_k=i, lse=f))}
    for name, (call, tensors) in calls.items():
        good = {k: on(t) for k, t in tensors.items()}
        with pytest.raises(AssertionError, match="was reached"):
            call(good)
        for k, t in tensors.items():
            with pytest.raises(mx.MxkError, match=f"{name}: .* on cpu"):
                call({**good, k: t})
            if k != "ws":
                with pytest.raises(mx.MxkError, match=f"{name}: .*{str(t.dtype)[6:]} belongs"):
                    call({**good, k: on(t.to(torch.int64 if t.dtype == torch.int32 else torch.float16))})
    cache._index = 1
    for name in ("qkv_norm_rope_append", "attn_decode_paged"):
        with pytest.raises(mx.MxkError, match=f"{name}: .* current device is cuda:0"):
            calls[name][0]({k: on(t) for k, t in calls[name][1].items()})
    with pytest.raises(mx.MxkError, match="attn_decode_workspace: .* current device is cuda:0"):
        mx.attn_decode_workspace(cache, 4)
    with pytest.raises(mx.MxkError, match="cu_q and cu_k"):
        mx.attn_window(on(bf), on(bf), on(bf), 4, 4, 4, 4, 64, 0.1, on(bf), cu_q=on(i), cu_k=on(i[:4]))
    with pytest.raises(mx.MxkError, match="AttnArgs"):
        mx.attn_window(on(bf), on(bf), on(bf), 4, 4, 1 << 32, 4, 64, 0.1, on(bf))


def test_plain_forms_of_the_benchmark_agree_with_the_reference():
    """The bounds of attention_ref hold for a softmax in 32 bits rounded once, and not for a wrong window."""
    import attention_ref as R
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, 64, generator=g).bfloat16() for n in (9, 33, 33))
    see = R.visible(9, 33, 5, 0, 2, "cpu")
    out, lse, bound, _ = R.attention_rows(q, k, v, 0.125, see)
    s = (0.125 * q.float() @ k.float().T).masked_fill(~see, float("-inf"))
    R.assert_within((s.softmax(1) @ v.float()).bfloat16(), out, bound)
    R.assert_within(s.logsumexp(1), lse, torch.full_like(lse, 1e-5))
    wrong = R.visible(9, 33, 6, 0, 2, "cpu")
    with pytest.raises(AssertionError):
        R.assert_within(R.attention_rows(q, k, v, 0.125, wrong)[0], out, bound)
