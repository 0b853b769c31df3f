"""What the token-paged cache and the rotary refuse or compute on the host, without a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import magi_b200 as mb
import paged_ref as R

L = mb._lib
E_BADARG, E_ALIGN, E_NOMEM = -1, -2, -5


class FakeCtx(C.Structure):
    """A context as the library lays it out, without a device behind it: enough for calls that are refused."""
    _fields_ = [("device", C.c_int), ("sm_count", C.c_int), ("workspace", C.c_void_p), ("err", C.c_char * 512)]


def cache(**kw):
    c = L.TokenCache()
    c.struct_size = C.sizeof(L.TokenCache)
    c.n_layers, c.n_pages, c.page_tokens, c.n_kv_heads, c.max_seqs, c.max_pages_per_seq = 1, 8, 16, 2, 4, 4
    for name in ("k8", "v8", "k_scale", "v_scale", "page_table", "seq_lens", "page_refs", "workspace"):
        setattr(c, name, 4096)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def ctx():
    return FakeCtx(0, 148, 4096, b"")


def test_struct_sizes_match_the_header(tmp_path):
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "magi_attn.h")
    mirror = {"magi_token_cache": L.TokenCache, "magi_paged_attn_params": L.PagedAttnParams, "magi_rotary_params": L.RotaryParams}
    body = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for s, m in mirror.items():
        body.append(f'printf("{s} . %zu\\n", sizeof({s}));')
        body += [f'printf("{s} {f[0]} %zu\\n", offsetof({s}, {f[0]}));' for f in m._fields_]
    (tmp_path / "p.c").write_text("\n".join(body + ["return 0;}"]))
    subprocess.check_call(["gcc", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")])
    for line in subprocess.check_output([str(tmp_path / "p")], text=True).split("\n"):
        if line:
            s, f, v = line.split()
            assert (C.sizeof(mirror[s]) if f == "." else getattr(mirror[s], f).offset) == int(v), line


@pytest.mark.parametrize("change,code", [(dict(struct_size=3), E_BADARG), (dict(page_tokens=48), E_BADARG), (dict(page_tokens=0), E_BADARG), (dict(n_layers=0), E_BADARG),
                                         (dict(n_pages=-1), E_BADARG), (dict(max_seqs=65537), E_NOMEM), (dict(n_pages=1 << 21), E_NOMEM), (dict(n_layers=1 << 24), E_NOMEM),
                                         (dict(max_pages_per_seq=1 << 28), E_NOMEM), (dict(n_kv_heads=65536), E_BADARG), (dict(k8=None), E_BADARG), (dict(page_refs=None), E_BADARG),
                                         (dict(v8=4104), E_ALIGN), (dict(workspace=4100), E_ALIGN)])
def test_a_bad_cache_is_refused_by_every_call(change, code):
    c, x = cache(**change), ctx()
    p = L.PagedAttnParams()
    p.struct_size = C.sizeof(L.PagedAttnParams)
    assert L.lib.magi_token_cache_reserve(C.byref(x), C.byref(c), 4096, 4096, 1, 4096, None) == code
    assert L.lib.magi_token_cache_append(C.byref(x), C.byref(c), 0, 4096, 4096, None, 1, 1, 1, 4096, 256, 128, 4096, 256, 128, None) == code
    assert L.lib.magi_token_cache_branch(C.byref(x), C.byref(c), 4096, 4096, 1, 1, None) == code
    assert L.lib.magi_token_cache_free(C.byref(x), C.byref(c), 4096, 1, None) == code
    assert L.lib.magi_token_cache_compact(C.byref(x), C.byref(c), None) == code
    assert L.lib.magi_paged_attn_fwd(C.byref(x), C.byref(c), C.byref(p), None) == code
    assert x.err


def test_null_contexts_and_caches():
    c = cache()
    assert L.lib.magi_token_cache_compact(None, C.byref(c), None) == E_BADARG
    assert L.lib.magi_token_cache_compact(C.byref(ctx()), None, None) == E_BADARG
    assert L.lib.magi_paged_attn_fwd(None, None, None, None) == E_BADARG
    assert L.lib.magi_rotary_fwd(None, None, None) == E_BADARG
    assert L.lib.magi_token_cache_workspace_bytes(0) == 0 and L.lib.magi_token_cache_workspace_bytes(10) >= 120


def test_bad_entries_are_refused():
    c, x = cache(), ctx()
    lib = L.lib
    assert lib.magi_token_cache_reserve(C.byref(x), C.byref(c), None, 4096, 1, 4096, None) == E_BADARG
    assert lib.magi_token_cache_reserve(C.byref(x), C.byref(c), 4096, 4096, -1, 4096, None) == E_BADARG
    assert lib.magi_token_cache_reserve(C.byref(x), C.byref(c), 4096, 4096, 1025, 4096, None) == E_NOMEM
    assert lib.magi_token_cache_reserve(C.byref(x), C.byref(c), 4096, 4096, 1, None, None) == E_BADARG
    assert lib.magi_token_cache_reserve(C.byref(x), C.byref(c), None, None, 0, None, None) == 0
    ok = (C.byref(x), C.byref(c), 0, 4096, 4096, 4096, 1, 1, 1, 4096, 256, 128, 4096, 256, 128, None)

    def append(**at):
        a = list(ok)
        for k, v in at.items():
            a[int(k[1:])] = v
        return lib.magi_token_cache_append(*a)

    assert append(_2=1) == E_BADARG and append(_2=-1) == E_BADARG and append(_7=-1) == E_BADARG and append(_8=-1) == E_BADARG
    assert append(_9=None) == E_BADARG and append(_9=4098) == E_ALIGN and append(_10=130) == E_ALIGN and append(_14=4) == E_ALIGN
    assert append(_5=None, _7=2) == E_BADARG and append(_5=None, _8=3) == E_BADARG
    assert append(_6=0) == 0 and append(_7=0) == 0


def test_attention_parameters_are_checked():
    def params(**kw):
        p = L.PagedAttnParams()
        p.struct_size = C.sizeof(L.PagedAttnParams)
        p.q = p.out = p.seqs = p.cu_q = p.workspace = 4096
        p.q_stride_t = p.o_stride_t = 512
        p.q_stride_h = p.o_stride_h = 128
        p.n, p.total_q, p.max_q, p.n_q_heads, p.causal = 1, 1, 1, 4, 1
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    c, x = cache(), ctx()
    for kw, code in ((dict(struct_size=1), E_BADARG), (dict(layer=1), E_BADARG), (dict(layer=-1), E_BADARG), (dict(n_q_heads=3), E_BADARG), (dict(n_q_heads=0), E_BADARG),
                     (dict(window=-1), E_BADARG), (dict(n=-1), E_BADARG), (dict(n=1025), E_NOMEM), (dict(cu_q=None, max_q=2), E_BADARG), (dict(cu_q=None, total_q=2), E_BADARG),
                     (dict(q=None), E_BADARG), (dict(workspace=None), E_BADARG), (dict(seqs=None), E_BADARG), (dict(q=4100), E_ALIGN), (dict(out=4104), E_ALIGN),
                     (dict(q_stride_t=516), E_ALIGN), (dict(n=0), 0), (dict(total_q=0), 0), (dict(max_q=0), 0)):
        assert L.lib.magi_paged_attn_fwd(C.byref(x), C.byref(c), C.byref(params(**kw)), None) == code, kw


def test_rotary_parameters_are_checked():
    def params(**kw):
        p = L.RotaryParams()
        p.struct_size = C.sizeof(L.RotaryParams)
        p.x = p.out = p.positions = p.inv_freq = 4096
        p.T, p.H, p.head_dim, p.rot_dim, p.dtype = 1, 1, 128, 64, L.DTYPE_F32
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    x = ctx()
    for kw, code in ((dict(struct_size=1), E_BADARG), (dict(dtype=1), E_BADARG), (dict(rot_dim=130), E_BADARG), (dict(rot_dim=7), E_BADARG), (dict(rot_dim=-2), E_BADARG),
                     (dict(H=0), E_BADARG), (dict(T=-1), E_BADARG), (dict(x=None), E_BADARG), (dict(inv_freq=None), E_BADARG), (dict(x=4097), E_ALIGN),
                     (dict(head_dim=8192, rot_dim=8192), E_BADARG), (dict(T=0), 0)):
        assert L.lib.magi_rotary_fwd(C.byref(x), C.byref(params(**kw)), None) == code, kw


def test_frequencies():
    plain, one = mb.rotary_frequencies(128, device="cpu")
    assert one == 1.0 and plain.dtype == torch.float64
    want = np.array([10000.0 ** (-2 * i / 128) for i in range(64)])
    assert np.allclose(plain.numpy(), want, rtol=1e-14)
    assert np.allclose(mb.rotary_frequencies(128, scaling="linear", factor=4.0, device="cpu")[0].numpy(), want / 4, rtol=1e-14)
    ntk = mb.rotary_frequencies(128, scaling="ntk", factor=8.0, device="cpu")[0].numpy()
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], want[-1] / 8, rel_tol=1e-12)   # fastest kept, slowest factor times slower
    yarn, m = mb.rotary_frequencies(128, scaling="yarn", factor=16.0, original_context=4096, device="cpu")
    ratio = yarn.numpy() / want
    turns = want * 4096 / (2 * math.pi)
    assert np.allclose(ratio[turns > 40], 1) and np.allclose(ratio[turns < 0.8], 1 / 16) and (np.diff(ratio) <= 1e-15).all()
    assert math.isclose(m, 0.1 * math.log(16) + 1)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.5), dict(rot_dim=8, scaling="x"), dict(rot_dim=8, scaling="yarn")):
        with pytest.raises(ValueError):
            mb.rotary_frequencies(device="cpu", **bad)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        mb.rotary(torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.float64))


def test_the_reference_quantiser_agrees_with_torch():
    """The tests' own e4m3 rounding against torch's cast, at every tie and end of the format."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(codes), np.isnan(R.CODES)) and np.array_equal(codes[~np.isnan(codes)], R.CODES[~np.isnan(R.CODES)])
    pos = R.CODES[:0x7f]
    ties = (pos[1:] + pos[:-1]) / 2
    y = np.concatenate([pos, ties, np.nextafter(ties, 0), np.nextafter(ties, 1e9), -ties, [0.0, 2.0 ** -10, 1e-30, 460.0]])
    y = y[np.abs(y) <= 448].astype(np.float32)
    assert np.array_equal(torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), R.to_code(y.astype(np.float64)))


def test_a_cache_without_its_use_counts_is_refused():
    for missing in ("page_uses", "scale_uses"):
        c, x = cache(page_uses=4096, scale_uses=4096), ctx()
        setattr(c, missing, None)
        assert L.lib.magi_token_cache_reserve(C.byref(x), C.byref(c), 4096, 4096, 1, 4096, None) == E_BADARG
        assert L.lib.magi_token_cache_append(C.byref(x), C.byref(c), 0, 4096, 4096, None, 1, 1, 1, 4096, 256, 128, 4096, 256, 128, None) == E_BADARG
        assert L.lib.magi_token_cache_branch(C.byref(x), C.byref(c), 4096, 4096, 1, 1, None) == E_BADARG
        assert L.lib.magi_token_cache_compact(C.byref(x), C.byref(c), None) == E_BADARG
        assert b"uses" in x.err


def test_scales_that_are_no_number_are_refused():
    c, x = cache(), ctx()
    for scale, code in ((math.nan, E_BADARG), (math.inf, E_BADARG), (2.5e38, E_BADARG), (2e38, 0), (1e-45, 0), (0.0, 0), (-1.0, 0), (-math.inf, 0)):
        p = L.PagedAttnParams()
        p.struct_size = C.sizeof(L.PagedAttnParams)
        p.n_q_heads, p.softmax_scale = 4, scale   # no entries: nothing runs
        p.cu_q = 4096
        assert L.lib.magi_paged_attn_fwd(C.byref(x), C.byref(c), C.byref(p), None) == code, scale


def test_views_that_share_memory_are_told_apart():
    """Against the sets of places themselves, for views of one buffer with the same strides; with others never too trusting."""
    from magi_b200.paged import _one_place_each, _overlap, _same_view
    rng = np.random.RandomState(0)
    buf = torch.zeros(4000, dtype=torch.float16)
    seen = {True: 0, False: 0}
    for i in range(4000):
        def view(shape=None, strides=None):
            shape = shape or (int(rng.randint(1, 6)), int(rng.randint(1, 5)), int(rng.randint(1, 9)))
            if strides is None:
                h = int(shape[2] + rng.randint(0, 6))
                strides = (int((shape[1] - 1) * h + shape[2] + rng.randint(0, 10)), h, 1)
                if rng.rand() < 0.3:   # heads outside
                    strides = (h, int((shape[0] - 1) * h + shape[2] + rng.randint(0, 10)), 1)
            return buf.as_strided(shape, strides, int(rng.randint(0, 300)))
        a = view()
        same = rng.rand() < 0.7
        b = view((int(a.shape[0] + rng.randint(0, 3)) if a.stride(0) >= a.stride(1) else a.shape[0],) + tuple(a.shape[1:]), a.stride()) if same else view(a.shape)
        try:
            _one_place_each(b, "b")
        except ValueError:   # a row more than its strides have room for: refused before
            continue
        places = [set((t.data_ptr() + 2 * (np.arange(t.shape[0])[:, None, None] * t.stride(0) + np.arange(t.shape[1])[:, None] * t.stride(1)
                                           + np.arange(t.shape[2]))).ravel().tolist()) for t in (a, b)]
        real = bool(places[0] & places[1])
        assert _overlap(a, b) == real if same else _overlap(a, b) >= real, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        seen[real] += 1
        if same and a.data_ptr() == b.data_ptr():
            assert _same_view(a, b)
    assert min(seen.values()) > 500
    assert not _overlap(buf[:0].view(0, 1, 1), buf.view(4000, 1, 1)) and _same_view(buf[:8].view(1, 1, 8), buf.as_strided((1, 1, 8), (3, 5, 1)))
    assert not _overlap(buf.view(4000, 1, 1), torch.zeros(4000, 1, 1, dtype=torch.float16))
