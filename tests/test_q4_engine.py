"""The inference engine over the 4-bit KV cache, with evictions, and the log-probabilities it records."""

import math

import pytest
import torch

from rl_project_b200.core.config import ModelSpec
from rl_project_b200.core.errors import ServingError
from rl_project_b200.inference import InferenceEngine, PagedQ4KVCache, SamplingParams
from rl_project_b200.models.transformer.model import TransformerLM

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def model(dev, n_embd=128, n_head=4, n_kv_head=2, block_size=256, **kw):
    torch.manual_seed(0)
    spec = ModelSpec(n_layer=2, n_head=n_head, n_kv_head=n_kv_head, n_embd=n_embd, block_size=block_size, dropout=0.0,
                     vocab_size=97, **kw)
    m = TransformerLM(spec).eval()
    return m.cuda().bfloat16() if dev == "cuda" else m


GREEDY = dict(temperature=0.0, top_k=None)
PROMPTS = [[1, 2, 3], list(range(5, 75)), [7] * 33, list(range(40, 57))]


@pytest.mark.parametrize("extra", [{}, {"sliding_window": 24, "alternating_layers": True, "attn_logit_cap": 30.0}])
def test_same_tokens_as_a_cache_of_rounded_rows(monkeypatch, extra):
    """The 4-bit engine generates what the plain cache does when every key and value is rounded on its way in."""
    from rl_project_b200.inference import engine as eng_mod
    from rl_project_b200.models.attention import causal
    from rl_project_b200.ops import paged_q4
    from rl_project_b200.ops.paged_attention import paged_write

    m = model("cpu", **extra)
    params = SamplingParams(max_tokens=20, **GREEDY)
    eng = InferenceEngine(m, max_batch=4, kv_cache="q4")
    assert isinstance(eng.kv, PagedQ4KVCache) and eng.kv.nbytes < 0.3 * InferenceEngine(m, max_batch=4).kv.nbytes
    got = [r.generated_tokens for r in eng.generate_batch(PROMPTS, params)]
    assert eng.allocator.used_blocks == 0

    def rounded(x):
        pools = [torch.zeros(-(-len(x) // 16), x.shape[1], paged_q4.q4_block_bytes(x.shape[2]), dtype=torch.uint8)
                 for _ in range(2)]
        at = torch.arange(len(x), dtype=torch.int32)
        paged_q4.paged_write_q4(x, x, *pools, at // 16, at % 16)
        return paged_q4._values(pools[0], x.shape[2]).transpose(1, 2).flatten(0, 1)[:len(x)]

    def write(k, v, k_pool, v_pool, blk, off, status=None):
        paged_write(rounded(k), rounded(v), k_pool, v_pool, blk, off)

    monkeypatch.setattr(causal, "paged_write", write)
    monkeypatch.setattr(eng_mod, "paged_write", write)
    ref = InferenceEngine(m, max_batch=4)
    assert [r.generated_tokens for r in ref.generate_batch(PROMPTS, params)] == got


@pytest.mark.parametrize("dev", DEVICES)
def test_evictions(dev):
    """Caches stay within the budget's bounds while positions go on; everything is returned at the end."""
    m = model(dev)
    eng = InferenceEngine(m, max_batch=4, kv_cache="q4", kv_budget=32, kv_sink=2, kv_recent=8)
    reqs = [eng.submit(p, SamplingParams(max_tokens=90, **GREEDY)) for p in PROMPTS]
    seen = {}
    while not all(r.finished for r in reqs):
        eng.step()
        for st in eng.states.values():
            n = len(st.req.generated_tokens)
            assert st.position == len(st.req.prompt_tokens) + n - 1
            if n > 2:
                assert st.cached <= 32 + 16
            seen[st.req.id] = max(seen.get(st.req.id, 0), st.evicted)
            assert len(eng.allocator.tables[st.req.id]) == -(-(st.cached + 1) // 16)
    assert all(len(r.generated_tokens) == 90 for r in reqs)
    # a prompt of 70 is cut to 32 at its second decode step at the latest, then after every 16 tokens
    by_prompt = {tuple(r.prompt_tokens): seen[r.id] for r in reqs}
    assert by_prompt[tuple(PROMPTS[1])] >= 70 + 88 - 48 and by_prompt[tuple(PROMPTS[0])] >= 3 + 88 - 48
    assert eng.stats()["evictions"] == eng.evictions > 8
    assert eng.allocator.used_blocks == (1 if eng.decode_graphs else 0)  # graph decode keeps a padding block
    assert sorted(eng._free_rows) == [0, 1, 2, 3]


@pytest.mark.parametrize("dev", DEVICES)
def test_cuts_by_weights_that_exist(monkeypatch, dev):
    """Every cut, a long prompt's first one too, follows the attention weights of the decode steps before it."""
    from rl_project_b200.ops import paged_q4

    cuts, evict = [], paged_q4.paged_evict_q4

    def spy(k_pool, v_pool, tables, lens, new, weights, rows, keep, head_dim, recent=0, sink=0, status=None):
        before = weights.clone()
        kept, left = evict(k_pool, v_pool, tables, lens, new, weights, rows, keep, head_dim, recent, sink, status)
        cuts.extend((before[int(r)].cpu(), int(n), kept[b].cpu()) for b, (r, n) in enumerate(zip(rows, lens)))
        return kept, left

    monkeypatch.setattr(paged_q4, "paged_evict_q4", spy)
    m = model(dev)
    eng = InferenceEngine(m, max_batch=2, kv_cache="q4", kv_budget=32, kv_sink=2, kv_recent=8)
    reqs = [eng.submit(p, SamplingParams(max_tokens=40, **GREEDY)) for p in (list(range(3, 73)) * 2, PROMPTS[2])]
    eng.step()
    assert not cuts and eng.evictions == 0  # prefilled and decoded once
    eng.step()
    assert len(cuts) == 2 and cuts[0][1] == 141  # (two layers; the short prompt has not grown enough yet)
    # one step of two query heads per KV head has weighed the prompt's tokens and its own
    assert ((cuts[0][0].sum(-1) - 2).abs() < 1e-2).all() and (cuts[0][0][:, 140] > 0).all()
    eng.run_until_idle()
    assert all(len(r.generated_tokens) == 40 for r in reqs) and len(cuts) > 8
    for row, n, kept in cuts:
        assert (row.sum(-1) > 1).all()
        for h in range(2):
            free = sorted(range(2, n - 8), key=lambda t: (-float(row[h, t]), t))[:22]
            assert kept[h].tolist() == sorted([0, 1] + free + list(range(n - 8, n)))


@pytest.mark.parametrize("dev", DEVICES)
def test_failed_eviction(monkeypatch, dev):
    """An eviction that raises fails the sequences that it was cutting, nobody else, and leaves no block behind."""
    eng = InferenceEngine(model(dev), max_batch=4, kv_cache="q4", kv_budget=32, kv_sink=2, kv_recent=8)
    evict = eng.kv.evict

    def fails_once(*args):
        monkeypatch.setattr(eng.kv, "evict", evict)
        raise RuntimeError("no eviction today")

    monkeypatch.setattr(eng.kv, "evict", fails_once)
    long, short = (eng.submit(p, SamplingParams(max_tokens=60, **GREEDY)) for p in (PROMPTS[1], PROMPTS[0]))
    eng.run_until_idle()
    assert long.finish_reason == "error" and "no eviction today" in long.error and len(long.generated_tokens) == 2
    assert len(short.generated_tokens) == 60 and short.finish_reason == "length" and eng.evictions > 0
    assert eng.allocator.used_blocks == (1 if eng.decode_graphs else 0) and sorted(eng._free_rows) == [0, 1, 2, 3]
    again = eng.generate(PROMPTS[1], SamplingParams(max_tokens=60, **GREEDY))
    assert again.finish_reason == "length" and len(again.generated_tokens) == 60


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("blocks", [15, 16, 19])
@pytest.mark.parametrize("same", [False, True])
def test_cuts_in_a_full_pool(dev, blocks, same):
    """Four sequences due in one step, in pools that hold them at their budget and one cut's copy, and little or nothing
    more: nobody fails for want of a block."""
    eng = InferenceEngine(model(dev), max_batch=4, kv_cache="q4", kv_budget=32, kv_sink=2, kv_recent=8,
                          max_blocks=blocks + (dev == "cuda"))  # (and the padding block)
    assert eng.allocator.reserve == 3 and eng.kv.num_blocks == blocks + (dev == "cuda")
    prompts = [[3 + i * (not same), 4, 5, 6] for i in range(4)]
    reqs = eng.generate_batch(prompts, SamplingParams(max_tokens=120, **GREEDY))
    assert [r.finish_reason for r in reqs] == ["length"] * 4 and all(len(r.generated_tokens) == 120 for r in reqs)
    assert eng.evictions >= 4 * 4 and eng.allocator.used_blocks == (1 if eng.decode_graphs else 0)


def test_request_ids_used_again():
    """A request under the id of one that still runs takes its place, as without a budget, and its accumulators' row."""
    for kw in ({}, {"kv_cache": "q4", "kv_budget": 32}):
        eng = InferenceEngine(model("cpu"), max_batch=2, **kw)
        for _ in range(5):
            last = eng.submit([1, 2, 3], SamplingParams(max_tokens=60, **GREEDY), id="same")
            eng.step()
        other = eng.submit([4, 5], SamplingParams(max_tokens=4, **GREEDY))
        eng.run_until_idle()
        assert len(last.generated_tokens) == 60 and len(other.generated_tokens) == 4
        assert sorted(eng._free_rows) == ([0, 1] if kw else [])


def test_blocks_kept_for_cuts():
    from rl_project_b200.inference import OutOfBlocksError, PagedBlockAllocator

    a = PagedBlockAllocator(block_size=4, max_blocks=6, reserve=2)
    a.allocate("a", 8)
    assert a.available == 2 and a.can_allocate("b", 8) and not a.can_allocate("b", 9)
    a.allocate("b", 8)
    with pytest.raises(OutOfBlocksError):
        a.append_token("a")
    assert a.lengths["a"] == 8
    old, new = a.replace("a", 5)
    assert not set(old) & set(new) and a.available == 0 and len(a.free_blocks) == 0
    a.release(old)
    assert a.available == 0 and len(a.free_blocks) == 2
    a.append_token("a")  # (its block has room)
    a.free("b")
    assert a.available == 2
    for bad in (6, -1):
        with pytest.raises(ServingError):
            PagedBlockAllocator(block_size=4, max_blocks=6, reserve=bad)
    with pytest.raises(ServingError):  # no block but the reserved ones
        InferenceEngine(model("cpu"), max_batch=1, kv_cache="q4", kv_budget=32, max_blocks=3)


def test_budget_never_reached_changes_nothing():
    m = model("cpu")
    params = SamplingParams(max_tokens=24, **GREEDY)
    outs = [[r.generated_tokens for r in InferenceEngine(m, max_batch=4, kv_cache="q4", **kw).generate_batch(PROMPTS, params)]
            for kw in ({}, {"kv_budget": 200})]
    assert outs[0] == outs[1]


@pytest.mark.parametrize("dev", DEVICES)
def test_shared_prompts_with_evictions(dev):
    """Samples of one prompt share its blocks until the first is cut; what it is cut from stays whole for the rest."""
    m = model(dev)
    prompt = list(range(3, 60))
    kw = dict(max_batch=4, kv_cache="q4", kv_budget=32, kv_sink=2, kv_recent=8)
    params = SamplingParams(max_tokens=40, **GREEDY)
    eng = InferenceEngine(m, **kw)
    reqs = [eng.submit(prompt, params) for _ in range(3)]
    eng.step()
    late = eng.submit(prompt, params)  # joins after the others were prefilled, maybe cut
    eng.run_until_idle()
    assert eng.shared_prefills >= 2
    alone = InferenceEngine(m, **kw).generate(prompt, params).generated_tokens
    if dev == "cpu":  # (bf16 products of another batch size round differently)
        assert all(r.generated_tokens == alone for r in reqs + [late])
    assert eng.allocator.used_blocks == (1 if eng.decode_graphs else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [None, 48])
@pytest.mark.parametrize("shape", [(256, 4, 1), (512, 4, 2), (128, 4, 4)])
def test_graph_decode_matches_eager_decode(shape, budget):
    """The same greedy requests decoded eagerly and from captured graphs, caches cut in between."""
    m = model("cuda", *shape)
    outs = {}
    for graphs in (False, True):
        eng = InferenceEngine(m, max_batch=8, decode_graphs=graphs, kv_cache="q4", kv_budget=budget)
        reqs = eng.generate_batch(PROMPTS, SamplingParams(max_tokens=60, **GREEDY))
        outs[graphs] = [r.generated_tokens for r in reqs]
        assert (eng.evictions > 3) == (budget is not None)
        if graphs:
            assert eng._graphs and eng.allocator.used_blocks == 1
    assert outs[True] == outs[False]
    from rl_project_b200.ops._ext import check_bounds

    check_bounds(torch.device("cuda", 0))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kv", ["bf16", "q4"])
def test_recorded_logprobs(dev, kv):
    """Log-probs and alternatives of every generated token, for the requests that ask for them."""
    m = model(dev)
    eng = InferenceEngine(m, max_batch=4, kv_cache=kv)
    asks = [3, None, 0, 20]
    reqs = [eng.submit(p, SamplingParams(max_tokens=6, temperature=t, top_k=None, logprobs=n))
            for p, n, t in zip(PROMPTS, asks, (0.0, 1.0, 1.0, 0.7))]
    eng.run_until_idle()
    for r, n in zip(reqs, asks):
        if n is None:
            assert not r.token_logprobs and not r.top_logprobs
            continue
        assert len(r.token_logprobs) == len(r.top_logprobs) == len(r.generated_tokens) == 6
        assert all(len(t) == n for t in r.top_logprobs)
        ids = torch.tensor([r.prompt_tokens + r.generated_tokens], device=dev)
        with torch.no_grad():
            want = m.full_logits(ids)[0].float().log_softmax(-1).cpu()
        # the model's own rounding (bf16 on the GPU, keys and values in 4 bits) moves log-probs; the first token's come
        # from the prompt's forward, which neither touches
        tol = {"cpu": {"bf16": 1e-3, "q4": 1.0}, "cuda": {"bf16": 0.15, "q4": 1.0}}[dev][kv]
        for i, tok in enumerate(r.generated_tokens):
            row = want[len(r.prompt_tokens) - 1 + i]
            bound = (1e-4 if dev == "cpu" else 0.1) if i == 0 else tol
            assert abs(r.token_logprobs[i] - float(row[tok])) <= bound
            top = r.top_logprobs[i]
            assert all(a[1] >= b[1] for a, b in zip(top, top[1:]))
            for t, lp in top:
                assert abs(lp - float(row[t])) <= bound
    assert [t[0][0] for t in reqs[0].top_logprobs] == reqs[0].generated_tokens  # greedy: the likeliest


def test_served_logprobs():
    from rl_project_b200.data.tokenizers import CharTokenizer
    from rl_project_b200.serving import EngineBackend, Router

    tok = CharTokenizer.ascii()
    torch.manual_seed(0)
    spec = ModelSpec(n_layer=1, n_head=2, n_kv_head=1, n_embd=64, block_size=128, dropout=0.0, vocab_size=tok.vocab_size)
    eng = InferenceEngine(TransformerLM(spec).eval(), max_batch=2, kv_cache="q4", kv_budget=16)
    router = Router({"m": EngineBackend("m", eng, tok, background=False)}, "m")
    status, out = router.handle("POST", "/v1/completions", {"prompt": "abc", "max_tokens": 30, "logprobs": 2})
    assert status == 200
    said, text = out["choices"][0]["logprobs"], out["choices"][0]["text"]
    assert "".join(said["tokens"]) == text and len(said["token_logprobs"]) == len(said["text_offset"]) == 30
    assert all(text[o:].startswith(t) for o, t in zip(said["text_offset"], said["tokens"]))
    assert all(len(t) == 2 for t in said["top_logprobs"]) and all(x <= 0 for x in said["token_logprobs"])
    stop = text[7]
    status, out = router.handle("POST", "/v1/chat/completions", {
        "messages": [{"role": "user", "content": "hi"}], "max_tokens": 5, "logprobs": True, "top_logprobs": 3})
    said = out["choices"][0]["logprobs"]["content"]
    assert status == 200 and len(said) == 5 and all(len(e["top_logprobs"]) == 3 for e in said)
    assert said[0]["bytes"] == list(said[0]["token"].encode())
    status, out = router.handle("POST", "/v1/completions", {"prompt": "abc", "max_tokens": 30, "temperature": 0,
                                                            "logprobs": 0, "stop": stop})
    said = out["choices"][0]["logprobs"]
    assert "".join(said["tokens"]) == out["choices"][0]["text"] and said["top_logprobs"] == [{}] * len(said["tokens"])
    status, out = router.handle("POST", "/v1/completions", {"prompt": "abc", "max_tokens": 3})
    assert out["choices"][0]["logprobs"] is None
    status, lines = router.handle("POST", "/v1/completions", {"prompt": "abc", "max_tokens": 3, "logprobs": 2, "stream": True})
    assert status == 200 and "[DONE]" in "".join(lines)
    for bad in ({"logprobs": 21}, {"logprobs": -1}, {"logprobs": "x"}, {"top_logprobs": 3}):
        assert router.handle("POST", "/v1/completions", {"prompt": "abc", **bad})[0] == 400


class Scripted:
    """An engine that answers every prompt with given tokens (all as likely as each other) and counts nothing else."""

    eos_token_id = None

    def __init__(self, tokens):
        self.tokens = tokens

    def submit(self, ids, params, **kw):
        from rl_project_b200.inference import GenerationRequest

        self.req = GenerationRequest(prompt_tokens=list(ids), params=params, **kw)
        self.req.start()
        for t in self.tokens:
            self.req.push_token(t, -1.0, [(t, -1.0)])
        self.req.finish("stop")
        return self.req

    def cancel(self, request_id):
        return True


def said_by(tokens, tokenizer, stop=()):
    from rl_project_b200.serving import EngineBackend

    return EngineBackend("m", Scripted(tokens), tokenizer, background=False).complete("x", SamplingParams(logprobs=1),
                                                                                     stop=stop)


def test_served_logprobs_of_every_token():
    """Bytes of one character and end marks that print nothing have their entries too."""
    from rl_project_b200.data.tokenizers import ByteTokenizer

    class WithEnd(ByteTokenizer):
        def decode(self, ids):
            return super().decode([i for i in ids if i != 0])

    for text in ("ab\U0001f600", "a\u00e9", "\u00e9b\U0001f600\U0001f600c"):
        for end in ([], [0], [0, 0]):
            ids = list(text.encode()) + end
            res = said_by(ids, WithEnd())
            assert res.text == text and res.completion_tokens == len(res.logprobs) == len(ids)
            offsets = [t.offset for t in res.logprobs]
            assert offsets == sorted(offsets) and all(0 <= o <= len(text) for o in offsets)
    assert len(said_by([0], WithEnd()).logprobs) == 1 and said_by([0], WithEnd()).text == ""
    res = said_by(list(b"abXcd"), WithEnd(), stop=("X",))  # cut at a stop string: what was cut off says nothing
    assert res.text == "ab" and [t.text for t in res.logprobs] == ["a", "b"]
    assert said_by(list(b"Xcd"), WithEnd(), stop=("X",)).logprobs == []


@pytest.mark.parametrize("stop", [(), ("\u00e9X",), ("never",)])
@pytest.mark.parametrize("path", ["/v1/completions", "/v1/chat/completions"])
def test_streamed_logprobs(path, stop):
    """A streamed answer's chunks carry, together, what the whole answer does."""
    import json

    from rl_project_b200.data.tokenizers import ByteTokenizer
    from rl_project_b200.serving import EngineBackend, Router

    class WithEnd(ByteTokenizer):
        def decode(self, ids):
            return super().decode([i for i in ids if i != 0])

    ids = list("n\U0001f600 a\u00e9\u00e9Xb\u00e9".encode()) + [0]
    router = Router({"m": EngineBackend("m", Scripted(ids), WithEnd(), background=False)}, "m")
    chat = "chat" in path
    body = {"prompt": "x", "messages": [{"role": "user", "content": "x"}], "stop": list(stop),
            **({"logprobs": True, "top_logprobs": 1} if chat else {"logprobs": 1})}
    whole = router.handle("POST", path, body)[1]["choices"][0]
    lines = list(router.handle("POST", path, {**body, "stream": True})[1])
    assert lines[-1] == "data: [DONE]\n\n"
    chunks = [json.loads(x[6:])["choices"][0] for x in lines[:-1]]
    text = whole["message"]["content"] if chat else whole["text"]
    assert "".join(c["delta"]["content"] if chat else c["text"] for c in chunks) == text
    assert len(chunks) > 4 and all("logprobs" in c for c in chunks[:-1]) and "logprobs" not in chunks[-1]
    for key, want in whole["logprobs"].items():
        assert [x for c in chunks[:-1] for x in c["logprobs"][key]] == want
    assert len(whole["logprobs"]["content" if chat else "tokens"]) == (
        len(text.encode()) + (stop != ("\u00e9X",)))  # (and the end mark, where the text was not cut)
    plain = [json.loads(x[6:])["choices"][0] for x in router.handle("POST", path, {
        "prompt": "x", "messages": body["messages"], "stream": True, "stop": list(stop)})[1] if "DONE" not in x]
    assert all("logprobs" not in c for c in plain)
    assert router.handle("POST", path, {**body, "stream": True, "logprobs": 21})[0] == 400


def test_offsets_in_linear_time():
    """A long answer's offsets, as its whole prefixes give them, from a number of decoded tokens in proportion to it."""
    from rl_project_b200.data.tokenizers import ByteTokenizer

    class Words:
        """Words with a leading space that the text's first word loses, as of some subword tokenizers; id 0 prints
        nothing."""

        seen = 0

        def encode(self, text):
            return [1]

        def decode(self, ids):
            Words.seen += len(ids)
            return "".join("" if i == 0 else " " + "w" * (int(i) % 5 + 1) for i in ids).removeprefix(" ")

    for end in (0, 30):
        ids = [(7 * i * i + i) % 23 for i in range(2000)] + [0] * end
        Words.seen = 0
        res = said_by(ids, Words())
        assert Words.seen <= 40 * len(ids)
        w = Words()
        assert [t.offset for t in res.logprobs] == [len(w.decode(ids[:i])) for i in range(len(ids))]
    text = "na\u00efve \U0001f600\u20ac " * 40
    res = said_by(list(text.encode()), ByteTokenizer())
    starts = [n for n, c in enumerate(text) for _ in c.encode()]
    assert [t.offset for t in res.logprobs] == starts and res.text == text
    broken = [0xff, 0x61, 0xf0, 0x9f, 0x98, 0x62] + [0xf0] * 9  # bytes that are no character: some offset, in order
    offsets = [t.offset for t in said_by(broken, ByteTokenizer()).logprobs]
    assert len(offsets) == len(broken) and offsets == sorted(offsets)


def test_alternatives_that_print_alike():
    """The completions answer names alternatives by their text: the likeliest of equal texts stays."""
    from rl_project_b200.serving.schemas import TokenLogprob, chat_response, completion_response

    top = [("\ufffd", -0.1), ("\ufffd", -3.0), ("b", -4.0)]
    said = [TokenLogprob("a", 0, -0.5, top)]
    out = completion_response("r", "m", "a", 1, 1, "length", logprobs=said)["choices"][0]["logprobs"]
    assert [list(t.items()) for t in out["top_logprobs"]] == [[("\ufffd", -0.1), ("b", -4.0)]]
    out = chat_response("r", "m", "a", 1, 1, "length", logprobs=said)["choices"][0]["logprobs"]["content"][0]
    assert [(e["token"], e["logprob"]) for e in out["top_logprobs"]] == top


def test_impossible_tokens_stay_within_json():
    import json

    from rl_project_b200.serving.schemas import TokenLogprob, chat_response, completion_response

    said = [TokenLogprob("a", 0, -0.5, [("b", -math.inf)]), TokenLogprob("c", 1, -math.inf, [])]
    for make in (chat_response, completion_response):
        json.dumps(make("r", "m", "ac", 1, 2, "length", logprobs=said), allow_nan=False)
    assert said[0].top == [("b", -9999.0)] and said[1].logprob == -9999.0 and said[0].logprob == -0.5


def test_no_number_stays_within_json():
    import json

    from rl_project_b200.serving.schemas import TokenLogprob, chat_response, completion_response

    said = [TokenLogprob("a", 0, math.nan, [("b", math.nan), ("c", math.inf), ("d", -math.inf), ("e", -0.25)])]
    for make in (chat_response, completion_response):
        json.dumps(make("r", "m", "a", 1, 1, "length", logprobs=said), allow_nan=False)
    assert said[0].logprob == -9999.0 and [x for _, x in said[0].top] == [-9999.0] * 3 + [-0.25]


def test_sink_fills_the_budget():
    """What the first tokens leave of the budget bounds the default share of the last ones."""
    m = model("cpu")
    eng = InferenceEngine(m, max_batch=2, kv_cache="q4", kv_budget=16, kv_sink=15)
    req, = eng.generate_batch([list(range(1, 41))], SamplingParams(max_tokens=30, **GREEDY))
    assert eng.kv_recent == 1 and eng.evictions > 0 and len(req.generated_tokens) == 30
    with pytest.raises(ServingError):
        InferenceEngine(m, kv_cache="q4", kv_budget=16, kv_sink=17)


@pytest.mark.parametrize("dev", DEVICES)
def test_prompts_written_by_table(dev):
    from rl_project_b200.inference import PagedQ4KVCache
    from rl_project_b200.ops.paged_q4 import paged_gather_q4

    kv = PagedQ4KVCache(2, 2, 32, 4, torch.device(dev))
    k, v = (torch.randint(0, 16, (2, 20, 32), device=dev).bfloat16() for _ in range(2))
    k[..., 0], k[..., 1], v[..., 0], v[..., 1] = 0, 15, 0, 15  # codes are the values
    kv.write_prefix(1, k, v, [3, 1])
    kv.copy_block(3, 0)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
    got = paged_gather_q4(*kv.layer(1), table, torch.tensor([20], dtype=torch.int32, device=dev), 32, 20)
    assert torch.equal(got[0][0].transpose(0, 1), k) and torch.equal(got[1][0].transpose(0, 1), v)
    assert not kv.k[0].any() and not kv.k[1, 2].any()


def test_refusals():
    m = model("cpu")
    for kw in ({"kv_cache": "int4"}, {"kv_budget": 64}, {"kv_cache": "q4", "kv_budget": 8},
               {"kv_cache": "q4", "kv_budget": 64, "kv_sink": 40, "kv_recent": 40},
               {"kv_cache": "q4", "kv_budget": 64, "kv_sink": -1}):
        with pytest.raises(ServingError):
            InferenceEngine(m, **kw)
    with pytest.raises(ServingError):  # heads of 16
        InferenceEngine(model("cpu", n_embd=64), kv_cache="q4")
    with pytest.raises(ServingError):  # windows count cached tokens
        InferenceEngine(model("cpu", sliding_window=24), kv_cache="q4", kv_budget=64)
    with pytest.raises(ServingError):
        SamplingParams(logprobs=21).validate()


def test_numbers_of_alternatives_are_whole():
    """A request that asks for 2.5 alternatives is refused alone; accepted, it would end the step of all the others."""
    import numpy as np

    eng = InferenceEngine(model("cpu"), max_batch=2)
    for bad in (2.5, float("nan"), True, "3", -1, 21):
        with pytest.raises(Exception) as err:
            eng.submit([1, 2], SamplingParams(max_tokens=2, logprobs=bad))
        assert isinstance(err.value, ServingError)
    req = eng.generate([1, 2], SamplingParams(max_tokens=2, logprobs=np.int64(2), **GREEDY))
    assert req.finish_reason == "length" and [len(t) for t in req.top_logprobs] == [2, 2]


def test_serve_sets_every_option_of_the_cache(monkeypatch):
    import importlib
    from types import SimpleNamespace

    from rl_project_b200.inference import engine as eng_mod

    cli, built = importlib.import_module("rl_project_b200.cli.main"), []

    class Engine(InferenceEngine):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            built.append(self)
            raise StopIteration

    monkeypatch.setattr(eng_mod, "InferenceEngine", Engine)
    monkeypatch.setattr(cli, "_load_policy", lambda args: SimpleNamespace(model=model("cpu"), tokenizer=None))
    for flags, want in (([], (64, 4, 16)), (["--kv-sink", "0", "--kv-recent", "30"], (64, 0, 30))):
        args = cli.build_parser().parse_args(["serve", "--checkpoint", "x", "--kv-cache", "q4", "--kv-budget", "64", *flags])
        with pytest.raises(StopIteration):
            cli.cmd_serve(args)
        assert (built[-1].kv_budget, built[-1].kv_sink, built[-1].kv_recent) == want


def test_rollouts_hold_their_cache_as_configured(monkeypatch):
    """engine_kv_cache reaches the engine of every rollout path, or is refused."""
    from types import SimpleNamespace

    import torch.distributed as dist

    from rl_project_b200.core.errors import RolloutError
    from rl_project_b200.parallel.runtime import free_port
    from rl_project_b200.rollouts import replicas
    from rl_project_b200.rollouts.engine import RolloutConfig, RolloutEngine
    from rl_project_b200.training.grpo import GRPOAlgorithm

    m = model("cpu")
    policy = SimpleNamespace(model=m, spec=m.spec, device=torch.device("cpu"))
    cfg = RolloutConfig(engine="paged", engine_kv_cache="q4", engine_max_batch=4, replica_tp=1)
    assert isinstance(RolloutEngine(policy, cfg).inference_engine().kv, PagedQ4KVCache)
    for name in ("generate", "auto"):  # no paged engine: on the CPU "auto" takes generate()
        other = RolloutConfig(engine=name, engine_kv_cache="q4")
        with pytest.raises(RolloutError):
            RolloutEngine(policy, other).inference_engine()
        assert RolloutEngine(policy, RolloutConfig(engine=name)).inference_engine() is None

    built = []

    class Replicas(replicas.RolloutReplicas):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            built.append(self.engine.kv)
            raise StopIteration

    monkeypatch.setattr(replicas, "RolloutReplicas", Replicas)
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{free_port()}", rank=0, world_size=1)
    try:
        with pytest.raises(StopIteration):
            GRPOAlgorithm._collect_replicated(SimpleNamespace(rollouts=RolloutEngine(policy, cfg), policy=policy,
                                                     _replica_set=None), 0)
    finally:
        dist.destroy_process_group()
    assert isinstance(built[0], PagedQ4KVCache)


def test_packed_scoring_through_logits():
    """The scoring path of policies that have logits only: values and gradients as from a plain log-softmax."""
    from types import SimpleNamespace

    from rl_project_b200.training.common.logprobs import pack_prompt_response, packed_response_logprobs

    torch.manual_seed(1)
    table = torch.randn(30, 30, requires_grad=True)
    policy = SimpleNamespace(pad_token_id=0, device=torch.device("cpu"), model=object(),
                             token_logits=lambda ids: table[ids])
    trajs = [SimpleNamespace(prompt_ids=torch.tensor(p), response_ids=torch.tensor(r))
             for p, r in (([1, 2], [3, 4, 5]), ([6], [7, 8]))]
    lp, ent = packed_response_logprobs(policy, trajs, 3, with_entropy=True)
    (lp[0].sum() + lp[1, :2].sum() + ent[0].sum() - ent[1, :2].sum()).backward()
    got, table.grad = table.grad, None
    inputs, targets = pack_prompt_response([([1, 2], [3, 4, 5]), ([6], [7, 8])], 0)
    logp = table[inputs].log_softmax(-1)
    want = logp.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    h = -(logp.exp() * logp).sum(-1)
    (want[0, 1:4].sum() + want[1, :2].sum() + h[0, 1:4].sum() - h[1, :2].sum()).backward()
    assert torch.allclose(lp[0], want[0, 1:4], atol=1e-5) and torch.allclose(ent[1, :2], h[1, :2], atol=1e-5)
    assert torch.allclose(got, table.grad, atol=1e-5) and math.isfinite(float(got.sum()))
