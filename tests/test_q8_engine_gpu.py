"""The engine with keys and values in 8 bits, sequences taken back, and both together with drafted tokens."""
import pytest
import torch

import furitar_cases
import plain_q8
import plain_qwen2 as P
from helpers import TOL, logits_err, make_folder, random_ids, rel_err

pytestmark = pytest.mark.gpu

LENGTHS = [37, 5, 90, 64, 130, 66]
# how the tokens behind each request's first part come: one, a few drafted ones, portions
CUTS = [1, 3, 1, 20, 1, 1, 5, 2, 40]
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def engine(folder, dtype, cache_dtype, max_tokens=2048, **more):
    from minfer_b200.engine.step import Engine
    from minfer_b200.model import Model
    return Engine(Model.from_folder(folder, dtype, "cuda:0"), max_tokens=max_tokens, cache_dtype=cache_dtype, **more)


def stored(eng, slot, layer, n):
    """(keys, values, their scales) [n, ...] float64 as the cache holds a sequence's first n positions."""
    g = eng.cache.group_of[layer]
    assert not g.ring or n <= g.ring
    (k, v), (ks, vs) = g.entry_tensors(layer), g.entry_scales(layer)
    out = []
    for codes, scales in ((k, ks), (v, vs)):
        c = torch.cat([codes[p].float().transpose(0, 1) for p in g.pages[slot]])[:n].cpu()
        s = torch.cat([scales[p].transpose(0, 1) for p in g.pages[slot]])[:n].cpu()
        out += [c.double() * s.double().unsqueeze(-1), s.double()]
    return out


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "F"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cache_dtype", list(FORMATS))
def test_against_the_plain_model(name, dtype, cache_dtype, monkeypatch):
    """Requests in a batch, their first parts as whole prompts, the rest cut in all ways, every place's
    logits.  The plain model attends, where the engine attends over its cache, over the keys and values the
    engine has stored, each of which must be its own key or value rounded to 8 bits."""
    folder = make_folder(name)
    cfg, w = P.load_folder(folder)
    prompts = [random_ids(n, cfg["vocab_size"], 100 + i) for i, n in enumerate(LENGTHS)]
    heads = [max(1, n // 2 - 3 * i) for i, n in enumerate(LENGTHS)]
    eng = engine(folder, dtype, cache_dtype)
    slots = [eng.acquire() for _ in prompts]
    got = [[] for _ in prompts]

    def step(rows, cuts):
        toks = [prompts[r][sum(len(x) for x in got[r]):][:c] for r, c in zip(rows, cuts)]
        out = eng.step([slots[r] for r in rows], toks, [list(range(len(t))) for t in toks])
        at = 0
        for r, t in zip(rows, toks):
            got[r].append(out[at:at + len(t)])
            at += len(t)

    step(list(range(len(prompts))), heads)
    turn = 0
    while True:
        rows = [r for r in range(len(prompts)) if sum(len(x) for x in got[r]) < LENGTHS[r]]
        if not rows:
            break
        if turn % 3 == 2:                                     # one token each: replayed steps
            step(rows, [1] * len(rows))
        else:
            step(rows, [CUTS[(turn + r) % len(CUTS)] for r in rows])
        turn += 1
    eng.check_status()
    eng.cache.check_canaries()
    fmt = FORMATS[cache_dtype]
    # float32: the engine's keys are off by TOL of the layer's largest; a code then by half a step
    slack = TOL[dtype]
    plain_attention = P.attention
    for r, ids in enumerate(prompts):
        layer = iter(range(cfg["num_hidden_layers"]))

        def attention(q, k, v, scale, window=0):
            k8, ks, v8, vs = stored(eng, slots[r], next(layer), len(ids))
            for have, scales, want in ((k8, ks, k), (v8, vs, v)):
                off = plain_q8.half_step(want, scales, fmt) * (1 + 2 * slack) + 2 * slack * want.abs().max()
                assert ((have - want).abs() <= off).all()
            whole = plain_attention(q, k, v, scale, window)[:heads[r]]
            return torch.cat([whole, plain_attention(q, k8.to(k.dtype), v8.to(v.dtype), scale, window)[heads[r]:]])

        monkeypatch.setattr(P, "attention", attention)
        want = P.forward(cfg, w, ids)
        monkeypatch.setattr(P, "attention", plain_attention)
        err, bound = logits_err(torch.cat(got[r]), want, dtype)
        assert err < bound, (name, r, err)


@pytest.mark.parametrize("dtype,name", [("float32", "B"), ("bfloat16", "D"), ("bfloat16", "E")])
def test_steps_through_graphs_equal_steps_kernel_by_kernel(dtype, name):
    folder = make_folder(name)
    vocab = P.load_folder(folder)[0]["vocab_size"]
    prompts = [random_ids(n, vocab, n) for n in (70, 3, 20)]
    outs = []
    for graphs in (True, False):
        eng = engine(folder, dtype, "e4m3", cuda_graphs=graphs)
        slots = [eng.acquire() for _ in prompts]
        eng.step(slots, prompts)
        rows = [eng.step(slots, [[(7 * i + j) % vocab] for j in range(3)]).clone() for i in range(12)]
        outs.append(torch.stack(rows))
        if graphs:
            assert eng._graphs
    assert rel_err(outs[0], outs[1]) < TOL[dtype]


@pytest.mark.parametrize("cache_dtype", [None, "e4m3", "int8"])
@pytest.mark.parametrize("dtype,name", [("float32", "A"), ("float32", "B"), ("bfloat16", "D")])
def test_taken_back_is_as_if_never_fed(dtype, name, cache_dtype):
    """A sequence is fed further, taken back and fed on: the same logits, bit for bit, as one that was never
    fed the rest (the step that follows has the same shape in both)."""
    folder = make_folder(name)
    vocab = P.load_folder(folder)[0]["vocab_size"]
    prompt, wrong, right = random_ids(60, vocab, 1), random_ids(90, vocab, 2), random_ids(9, vocab, 3)
    outs = []
    for detour in (False, True):
        eng = engine(folder, dtype, cache_dtype, cuda_graphs=False)
        other, s = eng.acquire(), eng.acquire()
        eng.step([other, s], [random_ids(64, vocab, 5), prompt])
        if detour:
            for cut in (wrong[:5], wrong[5:], [1]):
                eng.step([s], [cut])
                eng.rewind(s, len(prompt))
                assert eng.length(s) == len(prompt)
        rows = [eng.step([s], [right[:4]], [[0, 1, 2, 3]])] + [eng.step([s], [[t]]) for t in right[4:]]
        outs.append(torch.cat(rows))
        eng.check_status()
        eng.release(s)
        eng.release(other)
        assert all(n == g.n_pages for n, g in zip(eng.cache.free_pages(), eng.cache.groups))
    assert torch.equal(outs[0], outs[1])


def test_what_is_refused():
    from minfer_b200.engine.step import Engine, StepError
    from minfer_b200.model import Model
    model = Model.from_folder(furitar_cases.make_folder("A"), "float32", "cuda:0")
    with pytest.raises(StepError, match="activations' type only"):
        Engine(model, max_tokens=256, cache_dtype="int8")
    eng = Engine(model, max_tokens=256)
    s = eng.acquire()
    eng.step([s], [[1, 2, 3]])
    with pytest.raises(StepError, match="state"):
        eng.rewind(s, 2)
    folder = make_folder("B")                                 # a window of 16 in a ring of 128
    with pytest.raises(StepError, match="e4m3 or int8"):
        engine(folder, "float32", "fp4")
    eng = engine(folder, "float32", "int8", ring_step_tokens=100)
    s = eng.acquire()
    eng.step([s], [random_ids(200, 389, 1)])
    with pytest.raises(StepError, match="ring"):
        eng.rewind(s, 80)
    with pytest.raises(StepError, match="taken back"):
        eng.rewind(s, 201)
    eng.rewind(s, 190)
    eng.step([s], [[5]])
    eng.check_status()


def test_generation_and_the_command_line(tmp_path, capsys):
    """Greedy generation from an 8-bit cache: every token is the first choice of the step function over the
    same cache (kernel by kernel, fed one by one), and the command line gives the same."""
    from minfer_b200 import Generator, SamplingParams, cli
    from minfer_b200.model import Model
    folder = make_folder("D")
    vocab = P.load_folder(folder)[0]["vocab_size"]
    prompts = [random_ids(n, vocab, n) for n in (20, 70, 5)]
    model = Model.from_folder(folder, "float32", "cuda:0")
    got = Generator(model, max_tokens=1024, max_batch=4, cache_dtype="e4m3").generate(
        prompts, 12, SamplingParams.greedy(), stop_token_ids=[])
    for prompt, r in zip(prompts, got):
        eng = engine(folder, "float32", "e4m3", cuda_graphs=False)
        s = eng.acquire()
        logits = eng.step([s], [prompt])
        for t in r.tokens:
            top = float(logits.max())
            assert float(logits[0, t]) >= top - 1e-3 * float(logits.abs().max())
            logits = eng.step([s], [[t]])
    assert cli.main([folder, ",".join(map(str, prompts[0])), "--greedy", "-n", "12", "--dtype", "float32",
                     "--cache-dtype", "e4m3", "--n-ctx", "256"]) == 0
    assert " ".join(map(str, got[0].tokens)) in capsys.readouterr().out


@pytest.mark.parametrize("cache_dtype", ["e4m3", "int8", None])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("dtype,name", [("float32", "E"), ("bfloat16", "E"), ("bfloat16", "D")])
def test_drafted_tokens_over_the_cache(dtype, name, temperature, cache_dtype):
    """The operators as they are used together: a step of each row's last token and its drafts over the 8-bit
    cache, the verification of all rows, rows taken back to what was accepted.  Greedy: the tokens are
    those of steps of one token; drawn: accepted drafts and tokens are the plain verification's of the
    step's own logits."""
    from minfer_b200.kernels import api as K
    folder = make_folder(name)
    vocab = P.load_folder(folder)[0]["vocab_size"]
    gen = torch.Generator().manual_seed(3)
    prompts = [random_ids(n, vocab, n) for n in (30, 62, 5)]
    eng, one = engine(folder, dtype, cache_dtype), engine(folder, dtype, cache_dtype, cuda_graphs=False)
    slots, ones = [eng.acquire() for _ in prompts], [one.acquire() for _ in prompts]
    texts = [list(p) for p in prompts]
    first = eng.step(slots, prompts).argmax(-1).tolist()
    guide = one.step(ones, prompts)
    for t, x in zip(texts, first):
        t.append(x)
    for turn in range(7):
        # drafts: what steps of one token say, spoiled from some place on; none, one or several a row
        counts = [(turn + 2 * b) % 5 for b in range(3)]
        drafts = []
        for b, n in enumerate(counts):
            mine, keep = [], one.length(ones[b])
            feed = texts[b][keep:]
            for i in range(n):
                logits = one.step([ones[b]], [feed])[-1]
                x = int(logits.argmax())
                mine.append((x + 1) % vocab if (turn + b + i) % 4 == 3 else x)
                feed = [mine[-1]]
            drafts.append(mine)
            if one.length(ones[b]) > keep:
                one.rewind(ones[b], keep)
        start = [eng.length(s) for s in slots]
        logits = eng.step(slots, [[t[-1]] + d for t, d in zip(texts, drafts)], [list(range(n + 1)) for n in counts])
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        flat = [x for d in drafts for x in d]
        accept_u, draw_u = torch.rand(len(flat), generator=gen), torch.rand(3, generator=gen)
        accepted, tokens = (torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(2))
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        K.verify_drafts(logits, as_int(flat), as_int(cu), None, accept_u.cuda(), draw_u.cuda(), temperature, accepted,
                        tokens)
        got = accepted.tolist(), tokens.tolist()
        assert got == plain_q8.verify(logits.cpu().numpy(), flat, cu, None, accept_u.numpy(), draw_u.numpy(), temperature)
        for b, (n, x) in enumerate(zip(*got)):
            texts[b] += drafts[b][:n] + [x]
            eng.rewind(slots[b], start[b] + 1 + n)
            assert eng.length(slots[b]) == len(texts[b]) - 1
    eng.check_status()
    eng.cache.check_canaries()
    if temperature == 0.0:
        # (a code or a logit may turn on the last bit where a step has another shape: first choices are held
        # to the largest logit with that much room)
        room = {"float32": 1e-3, "bfloat16": 2 * TOL["bfloat16"]}[dtype]
        for b, t in enumerate(texts):
            n = len(prompts[b])
            one.rewind(ones[b], n)
            logits = guide[b]
            for x in t[n:]:
                assert float(logits[x]) >= float(logits.max()) - room * float(logits.abs().max())
                logits = one.step([ones[b]], [[x]])[0]
