"""The paged cache and rotary positions without a GPU: refusals, the host's account of pages, frequencies,
and the C ABI's argument checks."""

from __future__ import annotations

import ctypes
import math
import random
import re
import subprocess

import pytest
import torch

from conftest import ROOT

HEADER = ROOT / "include" / "pe_paged.h"


@pytest.fixture(scope="module")
def lib(pe):
    from packed_encoders_amd import _lib

    return _lib.library()


def test_header_and_binding_declare_the_same_entry_points(pe, lib):
    from packed_encoders_amd import _lib

    declared = set(re.findall(r"^int\s+(pe_\w+)\s*\(", HEADER.read_text(), flags=re.M))
    assert declared == set(_lib.PAGED_EXPORTED)
    assert all(hasattr(lib, name) for name in declared)


@pytest.mark.parametrize("struct,cname", [("PagedArgs", "pe_paged_args"), ("RotaryArgs", "pe_rotary_args"),
                                          ("AppendArgs", "pe_append_args")])
def test_ctypes_structs_match_the_header_layout(pe, tmp_path, struct, cname):
    import os
    import shutil

    from packed_encoders_amd import _lib

    gcc, hip_include = shutil.which("gcc"), "/opt/rocm/include"
    if gcc is None or not os.path.isdir(hip_include):
        pytest.skip("gcc or the HIP headers are not available")
    cls = getattr(_lib, struct)
    names = [f[0] for f in cls._fields_]
    body = "".join(f'    printf("%s %zu %zu\\n", "{n}", offsetof({cname}, {n}), sizeof((({cname} *)0)->{n}));\n'
                   for n in names)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "pe_paged.h"\nint main(void) {\n'
                   f'    printf("sizeof %zu 0\\n", sizeof({cname}));\n'
                   '    printf("macros %d %d\\n", PE_PAGED_PAGE_MULTIPLE, PE_PAGED_MAX_KEYS - PE_ROTARY_MAX_PAIRS);\n'
                   f'{body}    return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-D__HIP_PLATFORM_AMD__", "-I", str(ROOT / "include"), "-I", hip_include, str(src), "-o",
                    str(exe)], check=True, capture_output=True)
    got = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, off, size = line.split()
        got[name] = (int(off), int(size))
    assert got.pop("sizeof")[0] == ctypes.sizeof(cls)
    assert got.pop("macros") == (_lib.PAGE_MULTIPLE, _lib.PAGED_MAX_KEYS - _lib.ROTARY_MAX_PAIRS)
    assert got == {n: (getattr(cls, n).offset, getattr(cls, n).size) for n in names}


# ----------------------------------------------------------------------------- C argument checks


def _paged(**kw):
    from packed_encoders_amd import _lib

    a = _lib.PagedArgs()
    a.struct_size, a.dtype = ctypes.sizeof(a), _lib.DTYPE_BF16
    for name in ("q", "k_pages", "v_pages", "o", "page_table", "cu_seqlens", "seqlens_k"):
        setattr(a, name, 1 << 20)  # never read: every call here is refused, or only sized
    a.q_stride_token = a.o_stride_token = 4096
    a.q_stride_head = a.o_stride_head = a.k_stride_head = a.v_stride_head = 128
    a.k_stride_token = a.v_stride_token = 1024
    a.k_stride_page = a.v_stride_page = 1024 * 64
    a.n_seq, a.total_tokens, a.max_seqlen, a.max_seqlen_k = 4, 4, 1, 8192
    a.n_heads_q, a.n_heads_kv, a.head_dim = 32, 8, 128
    a.n_pages, a.page_size, a.max_pages, a.table_stride = 600, 64, 128, 128
    a.softmax_scale, a.window_left, a.window_right, a.causal = 0.1, -1, -1, 1
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,status", [
    ({"struct_size": 8}, -1), ({"dtype": 2}, -2), ({"n_seq": -1}, -1), ({"total_tokens": -1}, -1), ({"max_seqlen": -1}, -1),
    ({"max_seqlen_k": -1}, -1), ({"n_heads_kv": 3}, -1), ({"n_heads_kv": 0}, -1), ({"head_dim": 96}, -2),
    ({"softmax_scale": 0.0}, -1), ({"softmax_scale": math.nan}, -1), ({"softmax_scale": math.inf}, -1),
    ({"window_left": -2}, -1), ({"window_right": -2}, -1), ({"causal": 2}, -1), ({"page_size": 8}, -1),
    ({"page_size": 24}, -2), ({"page_size": 0}, -1), ({"n_pages": -1}, -1), ({"max_pages": -1}, -1),
    ({"table_stride": -1}, -1), ({"q": None}, -1), ({"o": None}, -1), ({"k_pages": None}, -1), ({"v_pages": None}, -1),
    ({"page_table": None}, -1), ({"cu_seqlens": None}, -1), ({"seqlens_k": None}, -1), ({"q": (1 << 20) + 8}, -1),
    ({"k_stride_token": 1028}, -1), ({"k_stride_token": 64}, -1), ({"v_stride_page": -8}, -1), ({"o_stride_token": 4}, -1),
    ({"max_seqlen_k": (1 << 29) + 1}, -2), ({"window_left": 1 << 30}, -2), ({"max_seqlen": 1 << 29}, -2), ({"k_stride_token": 1 << 26}, -2),
    ({"o_stride_token": 1 << 40}, -2), ({"o_stride_head": 1 << 40}, -2), ({"n_heads_q": 65544, "n_heads_kv": 8}, -2),
])
def test_attention_arguments_are_rejected_before_any_launch(lib, kw, status):
    assert lib.pe_paged_attn_fwd(ctypes.byref(_paged(**kw)), 1 << 20, 1 << 40, None) == status


def test_attention_needs_its_workspace(lib):
    size = ctypes.c_size_t(0)
    a = _paged()
    assert lib.pe_paged_workspace_size(ctypes.byref(a), ctypes.byref(size)) == 0
    assert 0 < size.value <= 256 << 20
    assert lib.pe_paged_attn_fwd(ctypes.byref(a), 1 << 20, size.value - 1, None) == -3
    assert lib.pe_paged_attn_fwd(ctypes.byref(a), None, size.value, None) == -3
    assert lib.pe_paged_attn_fwd(ctypes.byref(a), (1 << 20) + 4, size.value, None) == -3
    assert lib.pe_paged_workspace_size(ctypes.byref(a), None) == -1
    short = _paged(n_seq=1, total_tokens=1, max_seqlen_k=16)  # too few keys to spread
    assert lib.pe_paged_workspace_size(ctypes.byref(short), ctypes.byref(size)) == 0 and size.value == 0


def test_workspace_stays_bounded(lib):
    size = ctypes.c_size_t(0)
    for n, tokens, longest, keys in [(1, 1, 1, 1 << 29), (1, 4096, 4096, 1 << 20), (300, 300, 1, 1 << 17), (8, 60000, 9000, 9000),
                                    (40, 700, 300, 30000), (2, 33, 32, 1 << 20)]:
        for hq, hkv, d in [(32, 8, 128), (8, 2, 256), (64, 64, 256), (12, 12, 64), (48, 1, 256), (640, 640, 256), (9000, 9000, 64)]:
            a = _paged(n_seq=n, total_tokens=tokens, max_seqlen=longest, max_seqlen_k=keys, n_heads_q=hq, n_heads_kv=hkv,
                       head_dim=d)
            assert lib.pe_paged_workspace_size(ctypes.byref(a), ctypes.byref(size)) == 0
            assert size.value <= 256 << 20, (n, tokens, longest, keys, hq, hkv, d)


def test_empty_calls_launch_nothing(lib):
    assert lib.pe_paged_attn_fwd(ctypes.byref(_paged(n_seq=0, q=None)), None, 0, None) == 0
    assert lib.pe_paged_attn_fwd(ctypes.byref(_paged(total_tokens=0, q=None)), None, 0, None) == 0
    assert lib.pe_paged_attn_fwd(ctypes.byref(_paged(max_seqlen=0)), None, 0, None) == 0


def _rotary(**kw):
    from packed_encoders_amd import _lib

    a = _lib.RotaryArgs()
    a.struct_size, a.dtype = ctypes.sizeof(a), _lib.ROTARY_BF16
    a.x = a.out = a.positions = a.inv_freq = 1 << 20
    a.x_stride_token, a.x_stride_head, a.n_tokens, a.n_heads, a.head_dim, a.half, a.scale = 1024, 128, 4, 8, 128, 64, 1.0
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,status", [
    ({"struct_size": 8}, -1), ({"dtype": 0}, -2), ({"dtype": 4}, -2), ({"n_tokens": -1}, -1), ({"n_heads": -1}, -1),
    ({"head_dim": 0}, -1), ({"half": 0}, -1), ({"half": 65}, -1), ({"half": 257, "head_dim": 1024}, -2),
    ({"interleaved": 2}, -1), ({"inverse": -1}, -1), ({"positions_32": 3}, -1), ({"x": None}, -1), ({"out": None}, -1),
    ({"positions": None}, -1), ({"inv_freq": None}, -1), ({"x_stride_token": -8}, -1), ({"n_tokens": 1 << 40}, -2),
])
def test_rotary_arguments_are_rejected_before_any_launch(lib, kw, status):
    assert lib.pe_rotary_fwd(ctypes.byref(_rotary(**kw)), None) == status


def _append(**kw):
    from packed_encoders_amd import _lib

    a = _lib.AppendArgs()
    a.struct_size, a.dtype = ctypes.sizeof(a), _lib.DTYPE_BF16
    for name in ("q", "q_out", "k", "v", "k_pages", "v_pages", "page_table", "cu_seqlens", "seqlens_k", "inv_freq"):
        setattr(a, name, 1 << 20)
    a.q_stride_token, a.q_stride_head, a.k_stride_token, a.k_stride_head = 4096, 128, 2048, 128
    a.v_stride_token, a.v_stride_head = 2048, 128
    a.kp_stride_page = a.vp_stride_page = 65536
    a.kp_stride_token = a.vp_stride_token = 1024
    a.kp_stride_head = a.vp_stride_head = 128
    a.n_seq, a.total_tokens, a.n_heads_q, a.n_heads_kv, a.head_dim = 2, 5, 32, 8, 128
    a.n_pages, a.page_size, a.max_pages, a.table_stride, a.half, a.rope_scale = 100, 64, 8, 8, 64, 1.0
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,status", [
    ({"struct_size": 8}, -1), ({"dtype": 3}, -2), ({"n_seq": -1}, -1), ({"n_heads_kv": 0}, -1), ({"n_heads_q": 0}, -1),
    ({"q": None}, -1), ({"head_dim": 100, "half": 0}, -2), ({"half": 65}, -1), ({"half": -1}, -1), ({"interleaved": 2}, -1),
    ({"page_size": 20}, -2), ({"page_size": 1}, -1), ({"k": None}, -1), ({"v": None}, -1), ({"inv_freq": None}, -1),
    ({"q_out": None}, -1), ({"k_pages": None}, -1), ({"page_table": None}, -1), ({"v": (1 << 20) + 2}, -1),
    ({"kp_stride_token": 4}, -1), ({"vp_stride_page": -8}, -1), ({"n_heads_kv": 40000}, -2),
])
def test_append_arguments_are_rejected_before_any_launch(lib, kw, status):
    assert lib.pe_paged_append_fwd(ctypes.byref(_append(**kw)), None) == status


def test_page_copies_are_checked_on_the_host(lib):
    def call(src, dst, n_pages=8, page=64, stride=64, base=1 << 20):
        n = len(src)
        return lib.pe_copy_pages((ctypes.c_void_p * 1)(base), 1, stride, page, n_pages, (ctypes.c_int32 * n)(*src),
                                 (ctypes.c_int32 * n)(*dst), n, None)

    assert call([], []) == 0
    assert call([0], [8]) == -1 and call([-1], [0]) == -1 and call([8], [0]) == -1
    assert call([0, 1], [2, 2]) == -1  # a target twice
    assert call([0, 1], [1, 2]) == -1  # a target that is a source
    assert call([3], [3]) == -1
    assert call([0], [1], page=24) == -2 and call([0], [1], stride=72) == -2
    assert call([0], [1], page=128) == -1  # pages that overlap
    assert call([0], [1], base=(1 << 20) + 8) == -1


# ----------------------------------------------------------------------------- Python refusals


def test_calls_refuse_what_is_not_on_the_device(pe):
    q, pages = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    table, cu, lens = (torch.zeros(*s, dtype=torch.int32) for s in ((2, 1), (3,), (2,)))
    with pytest.raises(ValueError, match="HIP device"):
        pe.paged_attention(q, pages, pages.clone(), table, cu, lens, 1)
    with pytest.raises(ValueError, match="HIP device"):
        pe.paged_append(q[:, :2], q[:, 2:], pages, pages.clone(), table, cu, lens)
    with pytest.raises(ValueError, match="HIP device"):
        pe.copy_pages(pages, [0], [1])
    with pytest.raises(ValueError, match="HIP device"):
        pe.rotary(q, torch.zeros(2, dtype=torch.int64), torch.ones(8))
    with pytest.raises(ValueError, match="HIP device"):
        pe.rotary(q.requires_grad_(), torch.zeros(2, dtype=torch.int64), torch.ones(8))


def test_gradients_are_refused_where_there_are_none(pe):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="meta", requires_grad=True)
    pages = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    table, cu, lens = (torch.zeros(*s, dtype=torch.int32, device="meta") for s in ((2, 1), (3,), (2,)))
    with pytest.raises(ValueError, match="forward-only"):
        pe.paged_attention(q, pages, pages, table, cu, lens, 1)
    with pytest.raises(ValueError, match="forward-only"):
        pe.paged_append(q[:, :2], q[:, 2:], pages, pages, table, cu, lens)
    with torch.no_grad():
        assert pe.paged_attention(q, pages, pages, table, cu, lens, 1).shape == q.shape
        assert pe.paged_append(q[:, :2], q[:, 2:], pages, pages, table, cu, lens) is None
        assert pe.paged_append(q[:, :2], q[:, 2:], pages, pages, table, cu, lens, q=q).shape == q.shape


# ----------------------------------------------------------------------------- the host's account of pages


@pytest.fixture
def copies(pe, monkeypatch):
    """Page copies that a cache on no device asks for, in order."""
    from packed_encoders_amd import paged

    done = []
    monkeypatch.setattr(paged, "copy_pages", lambda pages, src, dst: done.append((list(src), list(dst))))
    return done


def _cache(pe, n_pages=16, page=16):
    return pe.PagedCache(2, n_pages, page, 2, 64, device="meta")


def test_sequences_take_and_return_pages(pe, copies):
    cache = _cache(pe)
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [17, 16])
    assert cache.pages(a) == (0, 1) and cache.pages(b) == (2,) and cache.free_pages == 13
    cache.extend([b], [1])
    assert len(cache.pages(b)) == 2 and cache.length(b) == 17
    cache.extend([a], [0])
    assert cache.length(a) == 17
    cache.close(a)
    assert cache.free_pages == 14 and not copies
    cache.truncate(b, 3)
    assert cache.pages(b) == (2,) and cache.length(b) == 3
    cache.truncate(b, 0)
    assert cache.pages(b) == () and cache.free_pages == 16
    with pytest.raises(ValueError):
        cache.truncate(b, 1)
    with pytest.raises(KeyError):
        cache.length(a)


def test_forks_share_pages_and_copy_a_last_page_once(pe, copies):
    cache = _cache(pe)
    a = cache.open()
    cache.extend([a], [20])
    kids = [cache.fork(a) for _ in range(3)]
    assert cache.free_pages == 14
    # all four write into the shared second page: three leave it, the last to come keeps it
    cache.extend([a, *kids], [1] * 4)
    (src, dst), = copies
    assert src == [1, 1, 1] and len(set(dst)) == 3 and not set(dst) & {0, 1}
    assert len({cache.pages(s)[1] for s in (a, *kids)}) == 4
    assert all(cache.pages(s)[0] == 0 for s in (a, *kids)) and cache.free_pages == 11
    cache.close(a)
    assert cache.free_pages == 12  # the first page still has users
    for s in kids:
        cache.close(s)
    assert cache.free_pages == 16


def test_unknown_sequences_change_nothing(pe, copies):
    cache = pe.PagedCache(1, 4, 16, 1, 64, device="cpu")
    for call in (cache.fork, cache.close, lambda s: cache.extend([s], [1]), lambda s: cache.truncate(s, 0)):
        with pytest.raises(KeyError):
            call(0)
    assert cache.free_pages == 4 and cache.open() == 0


def test_a_full_last_page_is_not_copied(pe, copies):
    cache = _cache(pe)
    a = cache.open()
    cache.extend([a], [32])
    b = cache.fork(a)
    cache.extend([a, b], [1, 2])
    assert not copies and cache.pages(a)[:2] == cache.pages(b)[:2] and cache.pages(a)[2] != cache.pages(b)[2]


def test_extend_changes_nothing_when_pages_run_out(pe, copies):
    cache = _cache(pe, n_pages=4)
    a = cache.open()
    cache.extend([a], [40])
    b = cache.fork(a)
    with pytest.raises(MemoryError):
        cache.extend([a, b], [1, 16])  # a copied page and a new one
    assert cache.length(a) == cache.length(b) == 40 and cache.pages(a) == cache.pages(b) and not copies
    with pytest.raises(ValueError):
        cache.extend([a, a], [1, 1])
    with pytest.raises(ValueError):
        cache.extend([a], [-1])
    with pytest.raises(KeyError):
        cache.extend([99], [1])
    cache.extend([b], [8])
    assert cache.free_pages == 0


def test_compaction_moves_the_highest_pages_down(pe, copies):
    cache = _cache(pe)
    seqs = [cache.open() for _ in range(4)]
    for s in seqs:
        cache.extend([s], [40])  # three pages each
    child = cache.fork(seqs[3])
    cache.close(seqs[0])
    cache.close(seqs[2])
    before = cache.pages(seqs[3])
    assert cache.compact() == 6
    (src, dst), = copies
    assert sorted(src) == [9, 10, 11] and sorted(dst) == [0, 1, 2]
    moved = dict(zip(src, dst))
    assert cache.pages(seqs[3]) == cache.pages(child) == tuple(moved[p] for p in before)
    assert cache.free_pages == 10 and cache.compact() == 6 and len(copies) == 1
    cache.extend([seqs[1]], [16])
    assert cache.pages(seqs[1])[3] == 6  # the lowest free page


def test_random_histories_keep_the_account(pe, copies):
    """Random opens, extensions, forks, truncations, closings and compactions against a plain model: contents
    by (sequence, position) follow the copies, no two sequences write one slot, every page is counted."""
    rng = random.Random(5)
    cache = _cache(pe, n_pages=40)
    model: dict[int, list[int]] = {}
    memory: dict[tuple[int, int], int] = {}  # (page, slot) -> token
    token = 0
    for _ in range(600):
        kind, seq = rng.random(), rng.choice(list(model) or [None])
        if seq is None or kind < 0.1:
            model[cache.open()] = []
        elif kind < 0.55:
            who = rng.sample(list(model), rng.randint(1, min(3, len(model))))
            counts = [rng.randint(0, 40) for _ in who]
            try:
                cache.extend(who, counts)
            except MemoryError:
                continue
            for src, dst in copies:
                for a, b in zip(src, dst):
                    memory.update({(b, t): memory[a, t] for t in range(16) if (a, t) in memory})
            copies.clear()
            written = set()
            for s, n in zip(who, counts):
                for _ in range(n):
                    at = len(model[s])
                    place = (cache.pages(s)[at // 16], at % 16)
                    assert place not in written
                    written.add(place)
                    memory[place] = token
                    model[s].append(token)
                    token += 1
        elif kind < 0.7:
            model[cache.fork(seq)] = list(model[seq])
        elif kind < 0.8:
            n = rng.randint(0, len(model[seq]))
            cache.truncate(seq, n)
            del model[seq][n:]
        elif kind < 0.9:
            cache.close(seq)
            del model[seq]
        else:
            used = cache.compact()
            for src, dst in copies:
                for a, b in zip(src, dst):
                    memory.update({(b, t): memory[a, t] for t in range(16) if (a, t) in memory})
            copies.clear()
            assert used == 40 - cache.free_pages and all(p < used for s in model for p in cache.pages(s))
        for s, tokens in model.items():
            assert cache.length(s) == len(tokens) and len(cache.pages(s)) == -(-len(tokens) // 16)
            assert [memory[cache.pages(s)[i // 16], i % 16] for i in range(len(tokens))] == tokens
        assert len({p for s in model for p in cache.pages(s)}) == 40 - cache.free_pages


def test_batch_builds_the_table(pe, copies):
    cache = pe.PagedCache(1, 8, 16, 1, 64, device="cpu")
    a, b, c = (cache.open() for _ in range(3))
    cache.extend([a, b], [33, 5])
    table, lens = cache.batch([b, a, c])
    assert table.tolist() == [[3, -1, -1], [0, 1, 2], [-1, -1, -1]] and lens.tolist() == [5, 33, 0]
    assert table.dtype == lens.dtype == torch.int32
    assert cache.batch([b], width=4)[0].tolist() == [[3, -1, -1, -1]]
    assert cache.batch([c])[0].shape == (1, 0)
    with pytest.raises(ValueError):
        cache.batch([a], width=2)


@pytest.mark.parametrize("kw", [{"layers": 0}, {"n_pages": 0}, {"page_size": 8}, {"page_size": 24}])
def test_cache_sizes_are_checked(pe, kw):
    sizes = {"layers": 1, "n_pages": 4, "page_size": 16, "n_heads_kv": 1, "head_dim": 64, **kw}
    with pytest.raises(ValueError):
        pe.PagedCache(**sizes, device="meta")


# ----------------------------------------------------------------------------- frequencies


def test_plain_frequencies(pe):
    inv, scale = pe.rotary_frequencies(8, 10000.0)
    want = [10000.0 ** (-2 * i / 8) for i in range(4)]
    assert inv.dtype == torch.float32 and scale == 1.0
    assert torch.equal(inv, torch.tensor(want, dtype=torch.float64).float())


@pytest.mark.parametrize("scaling,hf,extra", [
    ("linear", "linear", {}),
    ("ramp", "yarn", {"original_max_position_embeddings": 4096}),
    ("bands", "llama3", {"original_max_position_embeddings": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0}),
])
@pytest.mark.parametrize("dim,theta,factor", [(128, 500000.0, 8.0), (64, 10000.0, 4.0), (256, 160000.0, 2.0)])
def test_scaled_frequencies_match_transformers(pe, scaling, hf, extra, dim, theta, factor):
    """The same kinds of scaling as transformers computes them (in fp32, hence 1e-5)."""
    from types import SimpleNamespace

    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    params = {"rope_type": hf, "factor": factor, "rope_theta": theta, **extra}
    original = extra.get("original_max_position_embeddings", 4096)
    config = SimpleNamespace(head_dim=dim, hidden_size=dim * 4, num_attention_heads=4, rope_theta=theta,
                             max_position_embeddings=int(original * factor), rope_scaling=params,
                             rope_parameters=params, standardize_rope_params=lambda: None)
    want, want_scale = ROPE_INIT_FUNCTIONS[hf](config, "cpu")
    inv, scale = pe.rotary_frequencies(dim, theta, scaling=scaling, factor=factor, original=original)
    torch.testing.assert_close(inv, want.float(), rtol=1e-5, atol=0.0)
    assert abs(scale - want_scale) < 1e-6


def test_ntk_frequencies_end_where_they_should(pe):
    plain, _ = pe.rotary_frequencies(64, 10000.0)
    inv, scale = pe.rotary_frequencies(64, 10000.0, scaling="ntk", factor=4.0)
    assert inv[0] == 1.0 and scale == 1.0 and abs(float(plain[-1] / inv[-1]) - 4.0) < 1e-5


@pytest.mark.parametrize("args,kw", [((7, 1e4), {}), ((0, 1e4), {}), ((64, 0.0), {}), ((64, 1e4), {"factor": 0.5}),
                                     ((64, 1e4), {"scaling": "cubic"}), ((64, 1e4), {"scaling": "ramp", "factor": 2.0}),
                                     ((2, 1e4), {"scaling": "ntk", "factor": 2.0}),
                                     ((64, 1.0), {"scaling": "ramp", "original": 64}),
                                     ((64, 1e4), {"scaling": "ramp", "original": 64, "beta_slow": 0.0}),
                                     ((64, 1e4), {"scaling": "ramp", "original": 64, "beta_fast": 0.5}),
                                     ((64, 1e4), {"scaling": "bands", "original": 64, "low": 4.0})])
def test_frequency_refusals(pe, args, kw):
    with pytest.raises(ValueError):
        pe.rotary_frequencies(*args, **kw)
