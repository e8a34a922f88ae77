"""Paged KV cache without a GPU: what the entry points refuse, from Python and through the C ABI (a refused call launches
nothing, so no device is needed)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def paged():
    from qimeng_megakernel_b200 import _build
    _build.build()
    from qimeng_megakernel_b200 import paged
    return paged


i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)


def refused(exc, text, fn, *args, **kw):
    with pytest.raises(exc, match=text):
        fn(*args, **kw)


def test_block_tables_refusals(paged):
    f = paged.build_block_tables
    ok = dict(page_size=16, max_pages=4)
    refused(TypeError, "lengths must be a tensor", f, [1], i32(3), **ok)
    refused(TypeError, "lengths: expected torch.int32", f, i32(3).long(), i32(3), **ok)
    refused(ValueError, "lengths: expected 1 dim", f, i32(3, 1), i32(3), **ok)
    refused(ValueError, "lengths must be contiguous", f, i32(6)[::2], i32(3), **ok)
    refused(ValueError, "no requests", f, i32(0), i32(3), **ok)
    refused(ValueError, "page_size 24", f, i32(3), i32(3), page_size=24, max_pages=4)
    refused(ValueError, "max_pages 0", f, i32(3), i32(3), page_size=16, max_pages=0)
    refused(ValueError, "max_pages 1073741825", f, i32(3), i32(3), page_size=16, max_pages=2 ** 30 + 1)
    refused(ValueError, "1048577 requests", f, i32(2 ** 20 + 1), i32(3), **ok)
    refused(ValueError, "more than max_pages", f, i32(3), i32(3), prefix_table=i32(5), **ok)
    refused(ValueError, "out: expected", f, i32(3), i32(3), out=paged.BlockTables(i32(3, 5), i32(2)), **ok)
    refused(TypeError, "out.tables", f, i32(3), i32(3), out=paged.BlockTables(i32(3, 4).long(), i32(2)), **ok)
    refused(ValueError, "no CPU path", f, i32(3), i32(3), **ok)


def test_slot_map_refusals(paged):
    f = paged.build_slot_map
    ok = dict(page_size=16, tokens=4)
    refused(TypeError, "block_tables: expected", f, i32(3, 2).long(), i32(3), i32(3), **ok)
    refused(ValueError, "empty shape", f, i32(3, 0), i32(3), i32(3), **ok)
    refused(ValueError, "expected 3 requests", f, i32(3, 2), i32(2), i32(3), **ok)
    refused(ValueError, "expected 3 requests", f, i32(3, 2), i32(3), i32(4), **ok)
    refused(ValueError, "tokens 0", f, i32(3, 2), i32(3), i32(3), page_size=16, tokens=0)
    refused(ValueError, "tokens 16777217", f, i32(3, 2), i32(3), i32(3), page_size=16, tokens=2 ** 24 + 1)
    refused(ValueError, "1048577, 1", f, i32(2 ** 20 + 1, 1), i32(3), i32(3), **ok)
    refused(ValueError, "page_size 8", f, i32(3, 2), i32(3), i32(3), page_size=8, tokens=4)
    out = paged.SlotMap.empty(3, 4, "cpu")
    refused(ValueError, "out.slots: expected 5", f, i32(3, 2), i32(3), i32(3), page_size=16, tokens=5, out=out)
    refused(ValueError, "not be kv_lengths itself", f, i32(3, 2), out.kv_lengths, i32(3), out=out, **ok)
    refused(ValueError, "not be new_lengths itself", f, i32(3, 2), i32(3), out.kv_lengths, out=out, **ok)
    refused(ValueError, "no CPU path", f, i32(3, 2), i32(3), i32(3), out=out, **ok)


def attention(paged, T=3, H=8, HK=2, D=64, pages=6, page=16, seqs=2, room=4, prefix=32, **more):
    a = dict(q=bf(T, H, D), k=bf(pages, page, HK, D), v=bf(pages, page, HK, D), tables=i32(seqs, room), kv=i32(seqs),
             cu=i32(seqs + 1), prefix_table=i32(prefix // 16 if prefix >= 0 else 0), prefix_len=prefix)
    a.update(more)
    args = [a.pop(n) for n in ("q", "k", "v", "tables", "kv", "cu")]
    return paged.prefix_attention(*args, **a)


def test_attention_refusals(paged):
    f = lambda **kw: attention(paged, **kw)
    refused(TypeError, "q: expected torch.bfloat16", f, q=torch.zeros(3, 8, 64))
    refused(TypeError, "k_pages: expected torch.bfloat16", f, k=torch.zeros(6, 16, 2, 64).half())
    refused(ValueError, "q: expected .tokens, heads", f, q=bf(3, 512))
    refused(ValueError, "q: heads and dimensions", f, q=bf(3, 64, 8).transpose(1, 2))
    refused(ValueError, "16-byte aligned", f, q=bf(3 * 512 + 4)[4:].view(3, 8, 64))
    refused(ValueError, "head_dim 96", f, D=96)
    refused(ValueError, "head_dim 64 .cache 128", f, k=bf(6, 16, 2, 128), v=bf(6, 16, 2, 128))
    refused(ValueError, "k_pages .* differ", f, v=bf(5, 16, 2, 64))
    refused(ValueError, "query heads over", f, H=8, HK=3)
    refused(ValueError, "query heads over", f, H=17, HK=1)
    refused(ValueError, "k_pages must be contiguous", f, k=bf(6, 16, 4, 64)[:, :, :2])
    refused(ValueError, "page_size 48", f, page=48, prefix=48)
    refused(ValueError, "whole pages", f, prefix=24)
    refused(ValueError, "whole pages", f, prefix=-16)
    refused(ValueError, "at most 1073741824 positions", f, prefix_len=2 ** 31, prefix_table=i32(1))
    refused(ValueError, "67108865 pages of 16", f, tables=i32(1, 2 ** 26 + 1), kv=i32(1), cu=i32(2))
    refused(ValueError, "1048577 rows", f, q=bf(2 ** 20 + 1, 1, 64), k=bf(6, 16, 1, 64), v=bf(6, 16, 1, 64))
    refused(ValueError, "prefix_table has 1 pages", f, prefix_table=i32(1))
    refused(ValueError, "needs a prefix_table", f, prefix_table=None)
    refused(ValueError, "expected 1..1536 requests", f, seqs=1537)
    refused(ValueError, "expected kv_lengths", f, kv=i32(3))
    refused(ValueError, "expected kv_lengths", f, cu=i32(2))
    refused(ValueError, "scale 0", f, scale=0.0)
    refused(ValueError, "scale nan", f, scale=float("nan"))
    refused(ValueError, "scale inf", f, scale=float("inf"))
    refused(ValueError, "out: expected shape", f, out=bf(2, 8, 64))
    refused(ValueError, "lse: expected shape", f, lse=torch.zeros(3, 7))
    refused(TypeError, "lse: expected torch.float32", f, lse=bf(3, 8))
    refused(TypeError, "workspace: expected torch.uint8", f, workspace=torch.zeros(3))
    refused(RuntimeError, "no gradient", f, q=bf(3, 8, 64).requires_grad_())
    refused(RuntimeError, "no gradient", f, v=bf(6, 16, 2, 64).requires_grad_())
    refused(ValueError, "no CPU path", f)


def test_packed_arguments_match_the_structures(paged):
    from qimeng_megakernel_b200 import _lib
    for packed, structure in ((paged._TABLES, _lib.BlockTablesArgs), (paged._SLOTS, _lib.SlotMapArgs),
                              (paged._ATTENTION, _lib.PrefixAttentionArgs)):
        assert packed.size == C.sizeof(structure)
        values = [i + 1 for i in range(len(structure._fields_))]
        assert packed.pack(*values) == bytes(structure(*values))


def test_plan_walks_every_key_once(tmp_path):
    """The division of an attention call's work (tests/prefix_plan_sim.cpp includes the header the kernel is compiled with)."""
    exe = tmp_path / "prefix_plan_sim"
    subprocess.run(["g++", "-std=c++17", "-O2", "-o", str(exe), os.path.join(ROOT, "tests", "prefix_plan_sim.cpp")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert "prefix plan ok" in out.stdout


def test_c_entries_refuse_before_they_launch(paged):
    from qimeng_megakernel_b200 import _lib
    lib = _lib.load()
    assert lib.qmk_build_block_tables(None, 0, None) == -1
    assert lib.qmk_build_slot_map(None, 0, None) == -1
    assert lib.qmk_prefix_attention(None, 0, None) == -1
    P = 4096                                                       # an aligned address that nothing may touch

    def tables(**kw):
        a = dict(lengths=P, free_pages=P, prefix_table=P, tables=P, used=P, seqs=2, num_free=3, prefix_pages=1, page_size=16,
                 max_pages=4)
        a.update(kw)
        return lib.qmk_build_block_tables(bytes(_lib.BlockTablesArgs(**a)), 0, None)

    for kw in (dict(lengths=None), dict(tables=None), dict(used=None), dict(free_pages=None), dict(prefix_table=None),
               dict(seqs=0), dict(num_free=-1), dict(prefix_pages=-1), dict(page_size=0), dict(page_size=512),
               dict(page_size=17), dict(max_pages=0), dict(prefix_pages=5), dict(seqs=(1 << 20) + 1), dict(max_pages=(1 << 30) + 1)):
        assert tables(**kw) == -1, kw

    def slots(**kw):
        a = dict(block_tables=P, kv_lengths=P, new_lengths=P, slots=P, positions=P, seq_ids=P, active=P, cu_tokens=P,
                 kv_lengths_out=2 * P, seqs=2, tokens=3, page_size=16, max_pages=4)
        a.update(kw)
        return lib.qmk_build_slot_map(bytes(_lib.SlotMapArgs(**a)), 0, None)

    for name in ("block_tables", "kv_lengths", "new_lengths", "slots", "positions", "seq_ids", "active", "cu_tokens",
                 "kv_lengths_out"):
        assert slots(**{name: None}) == -1, name
    for kw in (dict(seqs=0), dict(tokens=0), dict(page_size=1), dict(max_pages=0), dict(kv_lengths=2 * P), dict(new_lengths=2 * P),
               dict(seqs=(1 << 20) + 1), dict(tokens=(1 << 24) + 1), dict(max_pages=(1 << 30) + 1)):
        assert slots(**kw) == -1, kw

    need = lib.qmk_prefix_attention_workspace(3, 2, 8, 2, 64, 32, 0)

    def attn(**kw):
        a = dict(q=P, out=P, lse=None, k_pages=P, v_pages=P, block_tables=P, kv_lengths=P, cu_tokens=P, prefix_table=P,
                 q_token_stride=512, out_token_stride=512, tokens=3, seqs=2, num_heads=8, num_kv_heads=2, head_dim=64,
                 page_size=16, num_pages=6, max_pages=4, prefix_len=32, scale=0.125, workspace=P,
                 workspace_bytes=max(need, 1 << 30))
        a.update(kw)
        return lib.qmk_prefix_attention(bytes(_lib.PrefixAttentionArgs(**a)), 0, None)

    for name in ("q", "out", "k_pages", "v_pages", "block_tables", "kv_lengths", "cu_tokens", "prefix_table"):
        assert attn(**{name: None}) == -1, name
    for kw in (dict(q=P + 8), dict(out=P + 2), dict(k_pages=P + 8), dict(v_pages=P + 8), dict(q_token_stride=508),
               dict(out_token_stride=516), dict(tokens=0), dict(seqs=0), dict(num_heads=9), dict(num_kv_heads=0),
               dict(num_heads=34), dict(seqs=1537), dict(tokens=(1 << 20) + 1), dict(head_dim=80), dict(num_pages=1 << 27),
               dict(max_pages=(1 << 26) + 1), dict(workspace=None), dict(workspace=P + 128), dict(page_size=48), dict(num_pages=0), dict(max_pages=0),
               dict(prefix_len=33), dict(prefix_len=-16), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attn(**kw) == -1, kw


def test_paged_step_refuses_without_a_handle(paged):
    from qimeng_megakernel_b200 import _lib
    lib = _lib.load()
    args = _lib.PagedStepArgs()
    assert lib.qmk_decode_step_paged(None, C.byref(args), None) == -1
    assert lib.qmk_paged_last_cuda_error() is not None


@pytest.mark.parametrize("batch,first,length,rows", [(3, 32, 70, 64), (1, 16, 20, 64), (40, 0, 30, 64), (2, 128, 150, 64),
                                                     (5, 64, 400, 64), (64, 0, 1, 64), (7, 5, 6, 8)])
def test_paged_prefill_plan(batch, first, length, rows):
    """Every sequence appends its tokens in order, no launch more than its rows."""
    from qimeng_megakernel_b200.prefill import paged_prefill_plan
    at = [first] * batch
    for s0, s1, positions in paged_prefill_plan(batch, first, length, rows):
        assert 0 < (s1 - s0) * len(positions) <= rows
        for s in range(s0, s1):
            assert positions == list(range(at[s], at[s] + len(positions)))
            at[s] += len(positions)
    assert at == [length] * batch


def test_paged_state_refusals(small_config, small_weights):
    from qimeng_megakernel_b200 import synthetic
    f = lambda **kw: synthetic.make_paged_globals(small_config, small_weights, **{**dict(prompt_len=20, max_new_tokens=4,
                                                  shared_prefix=16, batch=2, page_size=16, device="cpu"), **kw})
    refused(ValueError, "page_size 24", f, page_size=24)
    refused(ValueError, "keeps at least", f, shared_prefix=20)
    refused(ValueError, "keeps at least", f, shared_prefix=-1)
    refused(ValueError, "no CPU path", f)


def state(paged, seqs=2, room=4, rows=2, page=16, lengths=None, prefix_table=None, prefix_len=0, tables=None):
    return paged.PagedState(i32(seqs, room) if tables is None else tables, i32(seqs) if lengths is None else lengths, rows, page,
                            prefix_table, prefix_len)


def test_paged_state_looks_at_its_tables(paged):
    """What a state hands to the library as bare pointers has to be what the kernels read (int32, contiguous, long enough)."""
    f = lambda **kw: state(paged, **kw)
    refused(TypeError, "prefix_table: expected torch.int32", f, prefix_table=i32(2).long(), prefix_len=32)
    refused(ValueError, "prefix_table must be contiguous", f, prefix_table=i32(4)[::2], prefix_len=32)
    refused(ValueError, "prefix_table: expected 1 dim", f, prefix_table=i32(2, 1), prefix_len=32)
    refused(ValueError, "prefix_table has 1 pages", f, prefix_table=i32(1), prefix_len=32)
    refused(ValueError, "needs a prefix_table", f, prefix_len=16)
    refused(ValueError, "prefix_table is on meta", f, prefix_table=i32(2).to("meta"), prefix_len=32)
    refused(ValueError, "whole pages", f, prefix_table=i32(2), prefix_len=24)
    refused(ValueError, "whole pages", f, prefix_table=i32(2), prefix_len=-16)
    refused(TypeError, "block_tables: expected torch.int32", f, tables=i32(2, 4).long())
    refused(ValueError, "block_tables must be contiguous", f, tables=i32(4, 2).t())
    refused(ValueError, "block_tables: empty", f, tables=i32(0, 4), lengths=i32(0))
    refused(ValueError, "expected 1..1536 requests", f, seqs=1537)
    refused(ValueError, "lengths: expected", f, lengths=i32(1))
    refused(ValueError, "rows 0", f, rows=0)
    f(prefix_table=i32(3), prefix_len=32)


def test_a_replaced_table_is_looked_at_again(paged):
    """The kernel call's binding depends on every table of the state; what was put in one's place is checked again."""
    from qimeng_megakernel_b200 import mk_kernel
    s = state(paged, prefix_table=i32(2), prefix_len=32)
    s.check()
    for name, value in (("prefix_table", i32(3)), ("prefix_len", 16), ("block_tables", i32(2, 5))):
        before = mk_kernel._paged_sig(s)
        setattr(s, name, value)
        assert mk_kernel._paged_sig(s) != before, name
    s.check()
    s.prefix_table = i32(2).long()
    refused(TypeError, "prefix_table: expected torch.int32", s.check)
    s.prefix_table = i32(2)
    s.step.slots = i32(2)
    refused(TypeError, "step.slots: expected torch.int64", s.check)


def test_a_refused_step_leaves_the_state_as_it_was(paged):
    s = state(paged, lengths=torch.tensor([5, 9], dtype=torch.int32))
    for bad in (i32(3), i32(2).long(), i32(2), [1, 1]):                # (the third: no CPU path)
        with pytest.raises((TypeError, ValueError)):
            s.advance(bad)
        assert s.step.kv_lengths.tolist() == [5, 9]


def test_outputs_that_overlap_are_refused(paged):
    """Other CTAs still read what an output would write: an output that covers part of an input, or of another output, is refused."""
    from qimeng_megakernel_b200 import _lib
    lib = _lib.load()
    text = lambda: lib.qmk_paged_last_cuda_error().decode()

    def slots(**kw):                                               # 3 requests x 4 pages, 5 tokens, 4 KB apart
        a = {n: (i + 1) * 4096 for i, n in enumerate(("block_tables", "kv_lengths", "new_lengths", "slots", "positions", "seq_ids",
                                                      "active", "cu_tokens", "kv_lengths_out"))}
        a.update(seqs=3, tokens=5, page_size=16, max_pages=4)
        a.update({k: a[v[0]] + v[1] for k, v in kw.items()})
        return lib.qmk_build_slot_map(bytes(_lib.SlotMapArgs(**a)), 0, None)

    for kw in (dict(kv_lengths_out=("kv_lengths", 8)), dict(kv_lengths_out=("kv_lengths", -8)), dict(cu_tokens=("new_lengths", 0)),
               dict(cu_tokens=("kv_lengths", -12)), dict(kv_lengths_out=("new_lengths", 4)), dict(slots=("block_tables", 40)),
               dict(positions=("block_tables", -4)), dict(seq_ids=("positions", 16)), dict(active=("slots", 39)),
               dict(kv_lengths_out=("cu_tokens", 12)), dict(positions=("kv_lengths", 0))):
        assert slots(**kw) == -1, kw
        assert "overlap" in text(), kw

    def tables(**kw):                                              # 3 requests x 4 pages
        a = {n: (i + 1) * 4096 for i, n in enumerate(("lengths", "free_pages", "prefix_table", "tables", "used"))}
        a.update(seqs=3, num_free=6, prefix_pages=2, page_size=16, max_pages=4)
        a.update({k: a[v[0]] + v[1] for k, v in kw.items()})
        return lib.qmk_build_block_tables(bytes(_lib.BlockTablesArgs(**a)), 0, None)

    for kw in (dict(tables=("lengths", 8)), dict(used=("lengths", 8)), dict(tables=("free_pages", -44)), dict(prefix_table=("tables", 0)),
               dict(used=("tables", 44)), dict(used=("free_pages", 20))):
        assert tables(**kw) == -1, kw
        assert "overlap" in text(), kw
    assert lib.qmk_build_slot_map(None, 0, None) == -1 and text() == ""


def test_forward_mode_tangents_are_refused(paged):
    """A dual tensor's tangent would be dropped without a word."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        for name, shape in (("q", (3, 8, 64)), ("k", (6, 16, 2, 64)), ("v", (6, 16, 2, 64))):
            dual = forward_ad.make_dual(bf(*shape), bf(*shape))
            refused(RuntimeError, "no gradient", lambda: attention(paged, **{name: dual}))
            with torch.no_grad():                                  # (which does not stop forward mode)
                refused(RuntimeError, "no gradient", lambda: attention(paged, **{name: dual}))
        refused(ValueError, "no CPU path", lambda: attention(paged))


def test_scales_outside_32_bits_are_refused(paged):
    """The kernel multiplies by log2(e) * scale in 32 bits: a scale for which that is zero or infinite has no answer."""
    for scale in (1e39, 3e38, 1e-50):
        refused(ValueError, "scale .*: expected a positive number", lambda: attention(paged, scale=scale))
    for scale in (2e38, 1e-40, 1):
        refused(ValueError, "no CPU path", lambda: attention(paged, scale=scale))
    from qimeng_megakernel_b200 import _lib
    P = 4096
    a = dict(q=P, out=P, lse=None, k_pages=P, v_pages=P, block_tables=P, kv_lengths=P, cu_tokens=P, prefix_table=P, q_token_stride=512,
             out_token_stride=512, tokens=3, seqs=2, num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=6, max_pages=4,
             prefix_len=32, scale=3e38, workspace=P, workspace_bytes=1 << 30)
    assert _lib.load().qmk_prefix_attention(bytes(_lib.PrefixAttentionArgs(**a)), 0, None) == -1


def test_a_free_list_past_32_bits_is_refused(paged):
    free = torch.empty(1 << 31, dtype=torch.int32, device="meta")
    refused(ValueError, "free_pages: 2147483648 pages", paged.build_block_tables, i32(3), free, page_size=16, max_pages=4)
