"""Decode steps on the paged cache with a shared prefix against the contiguous cache: prefill, steps, the token loops, refusals.

Tolerances are those of the prefill tests of the batched kernel: the two routes round the attention's probabilities
differently (bf16 here, tf32 there), everything else is the same kernel."""
import pytest
import torch

from tests import _util as U

pytestmark = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _config(name):
    from qimeng_megakernel_b200.model_config import LLAMA_3_2_1B, OLMOE_1B_7B, QWEN3_0_6B
    base = {"llama": LLAMA_3_2_1B, "qwen3": QWEN3_0_6B, "olmoe": OLMOE_1B_7B}[name]
    return dict(base, num_hidden_layers=2, vocab_size=2048, max_position_embeddings=512)


def _prompts(cfg, batch, length, shared, seed):
    from qimeng_megakernel_b200 import synthetic
    prompts = synthetic.make_prompts(cfg["vocab_size"], batch, length, seed=seed)
    prompts[1:, :shared] = prompts[0, :shared]
    return prompts


def _dense_cache(g, name, layer, seq, length):
    """A sequence's rows of the pool, in order."""
    pages = g.paged.block_tables[seq].long()
    return getattr(g, name)[layer][pages].flatten(0, 1)[:length]


def _close(model, got, want, bound):
    """Rows (positions or sequences) within `bound`.  A token whose k-th and (k + 1)-th expert nearly tie may be routed to either:
    one of eight expert terms of about equal weight, all of independent random direction, is exchanged.  The expert sum
    (variance 8 t^2 of eight terms t) then moves by sqrt(2) t, half of itself, and the residual stream by that share of what the
    experts add to it; the mixture-of-experts tests bound such rows by 6e-2, and so does this one, for less than half of them."""
    got, want = got.float().flatten(1), want.float().flatten(1)
    err = (got - want).norm(dim=1) / want.norm(dim=1)
    if model == "olmoe":
        assert float(err.median()) <= bound and float(err.max()) <= 6e-2, err.tolist()
    else:
        assert float(err.max()) <= bound, err.tolist()


@pytest.mark.parametrize("model,batch,length,shared,page", [
    ("llama", 3, 70, 40, 16), ("llama", 1, 20, 16, 16), ("qwen3", 5, 100, 64, 32), ("olmoe", 4, 40, 17, 16),
    ("llama", 4, 30, 0, 64), ("qwen3", 2, 150, 128, 128)])
def test_paged_prefill_and_steps_match_the_contiguous_cache(model, batch, length, shared, page):
    _need_gpu()
    from qimeng_megakernel_b200 import synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config(model)
    weights = synthetic.make_weights(cfg, seed=11, device="cuda:0")
    prompts = _prompts(cfg, batch, length, shared, seed=40 + batch)
    steps = 5
    a = run_prefill_synthetic(cfg, weights, prompts, steps, shared_prefix=shared, page_size=page)
    b = run_prefill_synthetic(cfg, weights, prompts if batch > 1 else prompts[0], steps)
    assert a.globs.paged.prefix_len == shared // page * page
    for layer in range(2):
        for name in ("k_cache", "v_cache"):
            for s in range(batch):
                _close(model, _dense_cache(a.globs, name, layer, s, length), getattr(b.globs, name)[layer, s, :length], 1e-2)
    _close(model, a.logits, b.logits, 2e-2)
    # the same tokens through both, row by row the same logits
    ga, gb = a.globs, b.globs
    gen = torch.Generator().manual_seed(1)
    ga.token_in = torch.zeros(batch, dtype=torch.int64, device="cuda:0")
    gb.token_in = torch.zeros(batch, dtype=torch.int64, device="cuda:0")
    for i in range(steps):
        tok = torch.randint(0, cfg["vocab_size"], (batch,), generator=gen)
        ga.token_in.copy_(tok)
        gb.token_in.copy_(tok)
        ga.paged.advance()
        a.mk(ga)
        gb.position_id = length + i
        b.mk(gb)
        torch.cuda.synchronize()
        _close(model, ga.logits.view(batch, -1), gb.logits.view(batch, -1), 2e-2)
        la = ga.logits.view(batch, -1).float()
        assert ga.next_token.tolist() == la.argmax(-1).tolist()
        assert ga.paged.step.positions.tolist() == [length + i] * batch
    a.mk.check_status()
    b.mk.check_status()
    for x in (a, b):
        x.mk.close()


def test_token_loops_agree_on_the_paged_cache():
    """decode(): device loop, host loop and sampling with one candidate give the same tokens, and again the same."""
    _need_gpu()
    from qimeng_megakernel_b200 import synthetic
    from qimeng_megakernel_b200.decode import decode
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=3, device="cuda:0")
    prompts = _prompts(cfg, 4, 40, 33, seed=9)
    out = []
    for kw in (dict(), dict(decode_time=True), dict(host_loop=True), dict(temperature=1.0, top_k=1, seed=5)):
        pre = run_prefill_synthetic(cfg, weights, prompts, 12, shared_prefix=33, page_size=16)
        got = decode("llama-3.2-1b", prefill=pre, max_new_tokens=12, ignore_eos=True, **kw)
        out.append(got["new_tokens"].tolist())
        assert len(out[-1][0]) == 12 and pre.globs.paged.step.kv_lengths.tolist() == [40 + 11] * 4
        pre.mk.close()
    assert out[0] == out[1] == out[2]
    pre = run_prefill_synthetic(cfg, weights, prompts, 3, shared_prefix=33, page_size=16)
    with pytest.raises(ValueError, match="KV cache shorter"):
        decode("llama-3.2-1b", prefill=pre, max_new_tokens=30, ignore_eos=True)
    pre.mk.close()


@torch.inference_mode()
def test_finished_sequences_and_a_captured_step():
    """A step in which some sequences append nothing leaves their rows' places to the others; a captured step replays."""
    _need_gpu()
    from qimeng_megakernel_b200 import synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("qwen3")
    weights = synthetic.make_weights(cfg, seed=5, device="cuda:0")
    prompts = _prompts(cfg, 4, 50, 32, seed=21)
    pre = run_prefill_synthetic(cfg, weights, prompts, 8, shared_prefix=32, page_size=16)
    g, mk = pre.globs, pre.mk
    new = torch.tensor([1, 0, 1, 0], dtype=torch.int32, device="cuda:0")
    g.token_in = torch.tensor([5, 6, 0, 0], dtype=torch.int64, device="cuda:0")      # sequences 0 and 2
    lengths = g.paged.step.kv_lengths.clone()
    g.paged.advance(new)
    mk(g)
    mk.check_status()
    assert g.active_mask.tolist() == [1, 1, 0, 0] and g.kv_slots.tolist() == [0, 2, -1, -1]
    assert g.paged.step.kv_lengths.tolist() == [51, 50, 51, 50]
    pair = g.logits[:2].clone()
    assert (g.logits[2:].float() < -1e8).all()
    # the same step of all four, sequences 0 and 2 with the same tokens, from the same lengths
    g.paged.step.kv_lengths.copy_(lengths)
    g.token_in.copy_(torch.tensor([5, 9, 6, 9]))
    g.paged.advance()
    mk(g)
    torch.cuda.synchronize()
    full = g.logits.clone()
    assert U.rel_l2(full[[0, 2]], pair) <= 2e-2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.paged.step.kv_lengths.copy_(lengths)
        kept = g.paged.step.kv_lengths.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            g.paged.step.kv_lengths.copy_(kept)
            g.paged.advance()
            mk(g)
        g.logits.zero_()
        for _ in range(2):
            graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(g.logits, full)
    mk.check_status()
    mk.close()


@torch.inference_mode()
def test_rows_without_a_place_are_reported_and_calls_refused():
    _need_gpu()
    from qimeng_megakernel_b200 import _lib, mk_kernel, synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=6, device="cuda:0")
    prompts = _prompts(cfg, 2, 20, 16, seed=2)
    pre = run_prefill_synthetic(cfg, weights, prompts, 4, shared_prefix=16, page_size=16)
    g, mk = pre.globs, pre.mk
    g.token_in = torch.zeros(2, dtype=torch.int64, device="cuda:0")
    g.paged.advance()
    before = g.k_cache.clone()
    g.paged.step.slots[1] = 1 << 40                      # behind the pool: switched off, reported, nothing stored
    mk(g)
    with pytest.raises(_lib.QmkError):
        mk.check_status()
    assert (g.k_cache[:, 1:] != before[:, 1:]).any() and torch.isfinite(g.logits[0].float()).all()
    with pytest.raises(ValueError, match="slot map"):
        mk(g, 3)
    g.active_mask = g.active_mask.clone()
    with pytest.raises(ValueError, match="active_mask must be the buffer"):
        mk(g)
    mk.close()
    with pytest.raises(ValueError, match="differ within"):
        run_prefill_synthetic(cfg, weights, synthetic.make_prompts(cfg["vocab_size"], 2, 20, seed=2), 4, shared_prefix=16, page_size=16)
    with pytest.raises(ValueError, match="keeps at least"):
        run_prefill_synthetic(cfg, weights, prompts, 4, shared_prefix=20, page_size=16)
    with pytest.raises(ValueError, match="page_size 24"):
        run_prefill_synthetic(cfg, weights, prompts, 4, shared_prefix=16, page_size=24)
    mk_kernel.LlamaConfig.update_from_dict(cfg)


@torch.inference_mode()
def test_another_state_on_the_same_rows_and_the_contiguous_forms():
    """A PagedState put in the place of another one is looked over again; launches that know nothing of pages are refused."""
    _need_gpu()
    from qimeng_megakernel_b200 import paged, synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=6, device="cuda:0")
    pre = run_prefill_synthetic(cfg, weights, _prompts(cfg, 2, 20, 16, seed=2), 4, shared_prefix=16, page_size=16)
    g, mk = pre.globs, pre.mk
    g.token_in = torch.zeros(2, dtype=torch.int64, device="cuda:0")
    g.paged.advance()
    mk(g)
    host = torch.zeros(8, dtype=torch.int64)
    for call in (lambda: mk.generate_device(g, 20, 1), lambda: mk.generate_host(g, host, 0, 1), lambda: mk.run_phases(g, 0, 1),
                 lambda: mk.decode_step(20), lambda: mk.run_phases_bound(20, 0, 1)):
        with pytest.raises(ValueError, match="paged cache"):
            call()
    held = g.paged
    for rows in (1, 2):                                  # fewer rows than the step has; other buffers than the step reads
        g.paged = paged.PagedState(held.block_tables, held.step.kv_lengths, rows, 16, held.prefix_table, held.prefix_len)
        with pytest.raises(ValueError, match="1 rows" if rows == 1 else "must be the buffer"):
            mk(g)
    g.paged = held
    g.paged.advance()
    mk(g)
    mk.check_status()
    mk.close()


@torch.inference_mode()
def test_replays_of_a_captured_step_go_forward():
    """advance() and the kernel call captured once: every replay is the next step, as the same number of eager ones."""
    _need_gpu()
    from qimeng_megakernel_b200 import synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=5, device="cuda:0")
    prompts = _prompts(cfg, 3, 50, 32, seed=23)
    steps, seen = 7, []
    for captured in (False, True):
        pre = run_prefill_synthetic(cfg, weights, prompts, steps + 1, shared_prefix=32, page_size=16)
        g, mk = pre.globs, pre.mk
        g.token_in = pre.first_gen_token.view(-1).clone()
        g.next_token = g.token_in                        # the token a step picks is the next one's
        first = g.paged.step.kv_lengths
        g.paged.advance()                                # (an eager step before the capture)
        mk(g)
        rows = [[g.paged.step.positions.tolist(), g.paged.step.kv_lengths.tolist(), g.token_in.tolist()]]
        logits = [g.logits.clone()]
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                g.paged.advance()
                mk(g)
            assert g.paged.step.kv_lengths.tolist() == [51] * 3      # nothing has run
        for i in range(1, steps):
            if captured and i != 4:
                graph.replay()
            else:                                        # (eager steps in between go on where the replays were)
                g.paged.advance()
                mk(g)
            rows.append([g.paged.step.positions.tolist(), g.paged.step.kv_lengths.tolist(), g.token_in.tolist()])
            logits.append(g.logits.clone())
        mk.check_status()
        assert [r[0] for r in rows] == [[50 + i] * 3 for i in range(steps)]
        assert [r[1] for r in rows] == [[51 + i] * 3 for i in range(steps)]
        assert not captured or g.paged.step.kv_lengths.data_ptr() == first.data_ptr()
        seen.append((rows, logits))
        if captured:
            del graph
        mk.close()
    assert seen[0][0] == seen[1][0]
    assert all(torch.equal(a, b) for a, b in zip(seen[0][1], seen[1][1]))


def test_decode_starts_behind_the_prompt_every_time():
    """Several decode() calls on one prefill: each starts behind the prompt, as on the contiguous cache, whatever ran before."""
    _need_gpu()
    from qimeng_megakernel_b200 import synthetic
    from qimeng_megakernel_b200.decode import decode
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=3, device="cuda:0")
    prompts = _prompts(cfg, 4, 40, 33, seed=9)
    pre = run_prefill_synthetic(cfg, weights, prompts, 12, shared_prefix=33, page_size=16)
    run = lambda n, **kw: decode("llama-3.2-1b", prefill=pre, max_new_tokens=n, ignore_eos=True, **kw)["new_tokens"].tolist()
    first = run(12)
    assert run(12) == first and run(12, host_loop=True) == first
    assert [row[:5] for row in first] == run(5)
    pre.globs.paged.advance()
    assert run(12) == first and pre.globs.paged.step.kv_lengths.tolist() == [40 + 11] * 4
    with torch.inference_mode():
        pre.globs.paged.step.kv_lengths.copy_(torch.tensor([40, 39, 40, 40]))
    with pytest.raises(ValueError, match="fewer tokens than the prompt"):
        run(12)
    pre.mk.close()


@torch.inference_mode()
def test_a_token_without_a_page_is_reported():
    """A row whose token has no page (behind the table, or an entry of -1) is switched off, and the status says so; one that was
    switched off by hand is not reported."""
    _need_gpu()
    from qimeng_megakernel_b200 import _lib, synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=6, device="cuda:0")
    pre = run_prefill_synthetic(cfg, weights, _prompts(cfg, 2, 20, 16, seed=2), 4, shared_prefix=16, page_size=16)
    g, mk = pre.globs, pre.mk
    g.token_in = torch.tensor([3, 4], dtype=torch.int64, device="cuda:0")
    lengths = g.paged.step.kv_lengths.clone()
    g.paged.advance()
    mk(g)
    mk.check_status()
    good = g.logits.clone()
    # sequence 1 has no page for position 20
    g.paged.step.kv_lengths.copy_(lengths)
    page = g.paged.block_tables[1, 1].clone()
    g.paged.block_tables[1, 1] = -1
    g.paged.advance()
    mk(g)
    status = mk.poll_status()
    assert status["rc"] == -6 and status["code"] == 4 and status["detail"] == 1, status
    assert torch.equal(g.logits[0], good[0])
    mk.check_status()
    g.paged.block_tables[1, 1] = page
    # behind the table
    g.paged.step.kv_lengths.copy_(torch.tensor([20, 32]))
    g.paged.advance()
    mk(g)
    with pytest.raises(_lib.QmkError):
        mk.check_status()
    assert torch.equal(g.logits[0], good[0])
    # a sequence without a new token, and a row that the caller switched off, are nothing to report
    g.paged.step.kv_lengths.copy_(lengths)
    g.paged.advance(torch.tensor([1, 0], dtype=torch.int32, device="cuda:0"))
    mk(g)
    mk.check_status()
    g.paged.step.kv_lengths.copy_(lengths)
    g.paged.advance()
    g.active_mask[1] = 0
    mk(g)
    mk.check_status()
    assert torch.equal(g.logits[0], good[0])
    mk.close()


@torch.inference_mode()
def test_attention_failures_reach_the_status():
    """Offsets that do not ascend and a wait that runs out inside a step's attention: the rows are NaN, the status names it, and the
    next step is right."""
    _need_gpu()
    from qimeng_megakernel_b200 import _lib, synthetic
    from qimeng_megakernel_b200.prefill import run_prefill_synthetic
    cfg = _config("llama")
    weights = synthetic.make_weights(cfg, seed=6, device="cuda:0")
    # (a prefix: blocks and strips; none and short requests: strips alone)
    for shared in (32, 0):
        pre = run_prefill_synthetic(cfg, weights, _prompts(cfg, 3, 50, shared, seed=2), 6, shared_prefix=shared, page_size=16)
        g, mk = pre.globs, pre.mk
        g.token_in = torch.tensor([3, 4, 5], dtype=torch.int64, device="cuda:0")
        lengths = g.paged.step.kv_lengths.clone()
        g.paged.advance()
        mk(g)
        mk.check_status()
        good = g.logits.clone()
        g.paged.step.cu_tokens.copy_(torch.tensor([0, 2, 1, 3]))
        mk(g)
        status = mk.poll_status()
        assert status["rc"] == -6 and status["code"] == 5, status
        assert torch.isnan(g.attn_out.float()).all()
        g.paged.step.kv_lengths.copy_(lengths)
        g.paged.advance()
        mk(g)
        mk.check_status()
        assert torch.equal(g.logits, good)
        mk.set_timeout_cycles(20_000_000)                # about 10 ms
        mk.set_wait_first_dependency(True)               # the attention waits for a copy that nothing starts
        g.paged.step.kv_lengths.copy_(lengths)
        g.paged.advance()
        mk(g)
        status = mk.poll_status()
        mk.set_wait_first_dependency(False)
        mk.set_timeout_cycles(2_000_000_000)
        assert status["rc"] == _lib.ERR_DEVICE_TIMEOUT and status["code"] == 2 and status["phase"] == 1, status
        assert torch.isnan(g.attn_out.float()).all()
        g.paged.step.kv_lengths.copy_(lengths)
        g.paged.advance()
        mk(g)
        mk.check_status()
        assert torch.equal(g.logits, good)
        mk.close()
