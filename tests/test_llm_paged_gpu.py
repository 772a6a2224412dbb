"""Decoder over the paged cache against the same model over the contiguous one, and against itself: ragged batches, prompts
in chunks, captured steps, pages that run out.

Logits are compared with the bound of the contiguous harness test, 3e-2 of the largest one: between the two sides lie some
ten fp16 roundings a layer on the residual stream, in other orders, and fp16 against exact rotary angles.  An int8 row is off
by up to 1/254 of its largest value (4e-3) and an e4m3 row by 2^-4 of each (6e-2), in every cached key and value; errors of
independent rows average in the attention, so twice and five times the bound are allowed."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BOUND = 3e-2


@pytest.fixture(scope='module')
def model():
    import kairos_b200 as kb
    from kairos_b200 import llm, runtime
    cfg = llm.DecoderConfig('tiny', 2, 512, 8, 2, 64, 1024, 1000, 1e-5, 10000.0, True)
    kb.DynamicLinear.context = runtime.Context('cuda', cache_bytes=None)
    m = llm.Decoder(cfg, 'cuda')
    prof = kb.Profiler(m.linear_shapes())
    prof.load_table({s: [(4, 'w4a16_gemv'), (30000, 'w4a16_gemm')] for s in m.linear_shapes()})
    kb.DynamicLinear.prof = prof
    yield m
    kb.DynamicLinear.context = None
    kb.DynamicLinear.prof = None


def prompt(n, seed):
    return torch.randint(0, 1000, (n,), device='cuda', generator=torch.Generator('cuda').manual_seed(seed))


def steps(m, tokens, n, use_graph=True):
    out = []
    for i in range(n):
        m.tok.copy_(tokens[:, i:i + 1])
        m.decode_step(use_graph)
        out.append(m.logits.float().clone())
    return out


def close(a, b, factor=1.0):
    return (a.float() - b.float()).abs().max() <= factor * BOUND * b.float().abs().max()


@pytest.mark.parametrize('kv,factor', [('float16', 1.0), ('int8', 2.0), ('fp8_e4m3', 5.0)])
def test_paged_decoder_matches_the_contiguous_one(model, kv, factor):
    tokens = torch.stack([prompt(40, i) for i in range(3)])
    feed = torch.stack([prompt(12, 9 + i) for i in range(3)])
    model.allocate(3, 64)
    ref = [model.prefill(tokens, return_logits=True).clone()] + steps(model, feed, 12)
    model.allocate_paged(3, 64, kv, page_size=16)
    got = [model.prefill(tokens, return_logits=True).clone()] + steps(model, feed, 12)
    assert all(close(g, r, factor) for g, r in zip(got, ref))
    assert model.lens.tolist() == model.lengths == [52] * 3
    from kairos_b200 import runtime
    torch.cuda.synchronize()
    assert runtime.device_status() == 0


def test_ragged_batch_equals_its_sequences_alone(model):
    lens = [1, 33, 16, 50]
    feed = torch.stack([prompt(20, 30 + i) for i in range(4)])
    model.allocate_paged(4, 80, page_size=16)
    got = [model.prefill([prompt(n, n) for n in lens], return_logits=True).clone()] + steps(model, feed, 20)
    for i, n in enumerate(lens):
        model.allocate_paged(1, 80, page_size=32)
        ref = [model.prefill([prompt(n, n)], return_logits=True).clone()] + steps(model, feed[i:i + 1], 20)
        assert all(close(g[i:i + 1], r) for g, r in zip(got, ref))


@pytest.mark.parametrize('kv', ['float16', 'int8'])
def test_prompt_in_chunks_equals_the_whole_prompt(model, kv):
    whole = [prompt(61, 1), prompt(45, 2)]
    model.allocate_paged(2, 80, kv, page_size=16)
    ref = model.prefill(whole, return_logits=True).clone()
    model.prefill([whole[0][:20], whole[1][:3]])                 # a new prompt: the pages of the old one are used again
    assert model.lengths == [20, 3]
    model.prefill([whole[0][20:21], whole[1][3:40]], keep=True)
    got = model.prefill([whole[0][21:], whole[1][40:]], return_logits=True, keep=True)
    assert model.lengths == [61, 45]
    # the second pass sees the first one's keys as the cache holds them, as the whole prompt did too
    assert close(got, ref)


def test_captured_steps_equal_eager_ones(model):
    feed = torch.stack([prompt(40, 5), prompt(40, 6)])
    runs = []
    for graph in (False, True):
        model.allocate_paged(2, 80, page_size=16)
        model.prefill([prompt(7, 1), prompt(30, 2)])
        runs.append(steps(model, feed, 40, graph))               # crosses page borders: the table grows under the graph
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    out = model.generate([prompt(7, 1), prompt(30, 2)], 10)
    assert out.shape == (2, 10) and ((out >= 0) & (out < 1000)).all()


def test_pages_and_lengths_run_out_loudly(model):
    import kairos_b200 as kb
    model.allocate_paged(2, 64, page_size=16, num_pages=3)
    with pytest.raises(ValueError):
        model.prefill([prompt(3, 1)])
    with pytest.raises(ValueError):
        model.prefill([prompt(3, 1), prompt(0, 1)])
    with pytest.raises(ValueError):
        model.prefill([prompt(65, 1), prompt(3, 1)])
    model.prefill([prompt(31, 1), prompt(16, 1)])
    with pytest.raises(kb.KairosError):                          # the second sequence needs a fourth page
        model.decode_step()
    model.prefill([prompt(15, 1), prompt(15, 1)])
    ref = steps(model, torch.zeros((2, 1), dtype=torch.long, device='cuda'), 1)
    assert torch.isfinite(ref[0]).all()
    model.allocate(2, 64)
    with pytest.raises(ValueError):
        model.prefill(torch.stack([prompt(4, 1)] * 2), keep=True)


def test_a_refused_prompt_leaves_empty_sequences(model):
    import kairos_b200 as kb
    model.allocate_paged(2, 64, page_size=16, num_pages=3)
    model.prefill([prompt(20, 1), prompt(10, 2)])
    with pytest.raises(kb.KairosError):                          # the first prompt gets two pages, the second needs two
        model.prefill([prompt(32, 3), prompt(20, 4)])
    assert model.lengths == model.lens.tolist() == [0, 0]
    got = model.prefill([prompt(5, 5), prompt(32, 6)], return_logits=True).clone()      # fits once those are back
    assert model.paged.free_pages == 0
    model.allocate_paged(2, 64, page_size=16)
    assert close(got, model.prefill([prompt(5, 5), prompt(32, 6)], return_logits=True))


def test_measurements_say_how_the_prefill_ran(model):
    from kairos_b200 import llm
    short = dict(prompt_len=8, new_tokens=3, warmup=1, ttft_times=1)
    for kw, want, graphs in ((dict(), 'graph', 1), (dict(prefill_graph=False), 'eager', 0), (dict(kv_dtype='int8'), 'eager', 0)):
        assert llm.measure_ttft_tpot(model, 2, **short, **kw)['prefill'] == want
        assert len(model._prefill_graphs) == graphs


@pytest.mark.parametrize('paged', [False, True])
def test_logits_are_those_of_the_last_step(model, paged):
    """Captured and eager steps in turn: the logits follow whichever ran last."""
    feed = torch.stack([prompt(8, 5), prompt(8, 6)])
    runs = []
    for modes in ([False] * 8, [True, False, True, True, False, False, True, True]):
        model.allocate_paged(2, 32, page_size=16) if paged else model.allocate(2, 32)
        model.prefill(torch.stack([prompt(7, 1), prompt(7, 2)]))
        out = []
        for i, graph in enumerate(modes):
            out += steps(model, feed[:, i:i + 1], 1, graph)
            assert torch.equal(model.next_tok[:, 0], out[-1].argmax(-1))
        runs.append(out)
    assert all(close(a, b) for a, b in zip(*runs))
