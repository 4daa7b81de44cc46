"""BatchDecoder (several sequences over a paged cache) and the serving options
of PFlashDecoder on the small model of tests/decode_model.py (2 layers, 4/2
heads of 64), against its fp32 restatement.

Tolerance of the logits (normwise): an attention with fp16 operands rounds q,
k, v, the weights and the output once each, half a step 2^-11 relative, 2.5e-3
in all; each of the two layers adds it to a residual stream that is larger
than the attention's part, and norms, linears and the lm_head pass a relative
error on: 2 * 2.5e-3, doubled for the growth through the SwiGLU product: 1e-2.
bf16's half step is eight times that."""
import pytest
import torch

import decode_model as dm
from polarflash_b200.batch import PageAllocator

gpu = pytest.mark.gpu
CFG = dm.CFG


def test_page_allocator():
    a = PageAllocator(5)
    x, y = a.take(3), a.take(2)
    assert sorted(x + y) == list(range(5)) and len(a) == 0
    with pytest.raises(RuntimeError):
        a.take(1)
    a.give(x)
    assert len(a) == 3 and sorted(a.take(3)) == sorted(x)
    assert a.take(0) == []


def test_prompt_dtype_is_refused_for_heads_it_does_not_take():
    from polarflash_b200.decode import PFlashDecoder

    for hd in (136, 20):
        cfg = dict(CFG, hidden_size=4 * hd)
        x = torch.zeros(CFG["vocab_size"], 4 * hd)
        args = (cfg, [], x, x[0], x, 8)
        PFlashDecoder(*args)
        with pytest.raises(ValueError):
            PFlashDecoder(*args, prompt_dtype=torch.bfloat16)


def _parts():
    from test_decode_step import _decoder

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    w = dm.build()
    d = _decoder(w, max_seq=64)
    return w, d


def _batch(d, **kw):
    from polarflash_b200 import BatchDecoder

    args = dict(max_seqs=4, max_seq=64, num_pages=12, page_size=16, kv_mode="fp16", prompt_dtype=torch.float16)
    args.update(kw)
    return BatchDecoder(CFG, d.layers, d.embed, d.final_norm, d.lm_head, **args)


def _rel(a, b):
    return float((a.double().cpu() - b.double().cpu()).abs().max() / b.double().cpu().abs().max())


PROMPTS = [dm.PROMPT, dm.PROMPT[:7], [300], dm.PROMPT[3:19]]
TOKENS = [[11, 300, 64], [5, 9, 200], [1, 2, 3], [250, 0, 383]]


@gpu
@pytest.mark.parametrize("mode,dt,tol", [("fp16", torch.float16, 1e-2), ("bf16", torch.bfloat16, 8e-2), ("int8", torch.float16, 1e-2)])
@pytest.mark.parametrize("graph", [False, True])
def test_batch_decoder_matches_single_sequences(mode, dt, tol, graph):
    """Prompts of 20, 7, 1 and 16 tokens (a page ends with the last), three steps
    over page borders.  int8: the restatement's cache is quantized behind the
    prompt and with every step, as the pages are."""
    from polarflash_b200.kv_cache import kv_dequantize, kv_quantize

    w, d = _parts()
    b = _batch(d, kv_mode=mode, prompt_dtype=dt)
    if graph:
        b.capture()
    slots, logits = b.add([torch.tensor(p) for p in PROMPTS])
    assert slots == [0, 1, 2, 3] and logits.shape == (4, CFG["vocab_size"])

    def quant(x):
        c, s, z = kv_quantize(x.cuda(), "int8")
        return kv_dequantize(c, s, z, x.shape[-1], "int8").cpu()

    caches = []
    for i, p in enumerate(PROMPTS):
        caches.append([{} for _ in range(CFG["num_hidden_layers"])])
        assert _rel(logits[i], dm.reference_forward(w, p, caches[i])[-1]) < tol
        if mode == "int8":
            for c in caches[i]:
                c["k"], c["v"] = quant(c["k"]), quant(c["v"])
    for t in range(3):
        tok = torch.tensor([TOKENS[i][t] for i in range(4)], device="cuda")
        got = b.step(tok)
        for i in range(4):
            ref = dm.reference_forward(w, [TOKENS[i][t]], caches[i], kv_quant=quant if mode == "int8" else None)[-1]
            assert _rel(got[i], ref) < tol, (t, i)
    assert b.lengths == [23, 10, 4, 19]


@gpu
def test_batch_decoder_slots_and_pages():
    """A sequence's logits do not depend on its slot, its pages or the other
    sequences; released pages are used again; calls that cannot be served are
    refused and change nothing."""
    _, d = _parts()
    b = _batch(d)
    p = [torch.tensor(x) for x in PROMPTS]
    tok = torch.tensor([11, 12, 13, 14], device="cuda")
    slots, first = b.add([p[0]])
    one = b.step(tok).clone()[slots[0]]
    free = len(b.allocator)
    assert free == 12 - 2
    s2, _ = b.add([p[1], p[2]])
    assert s2 == [1, 2] and b.active() == [0, 1, 2]
    b.step(tok)
    b.release(0)
    assert b.active() == [1, 2] and len(b.allocator) == 12 - 2
    s3, again = b.add([p[3], p[0]])
    assert s3 == [0, 3]
    assert _rel(again[1], first[0]) < 1e-4  # the GEMMs of another batch size
    got = b.step(torch.tensor([7, 5, 5, 11], device="cuda"))[3]
    assert _rel(got, one) < 1e-4
    state = (list(b.lengths), len(b.allocator), b._table.clone(), b._lens.clone())
    for bad in ([], [torch.tensor([], dtype=torch.long)], [torch.zeros(65, dtype=torch.long)], [torch.tensor([CFG["vocab_size"]])],
                [torch.tensor([-1])]):
        with pytest.raises((ValueError, RuntimeError)):
            b.add(bad)
    with pytest.raises(RuntimeError):
        b.add([p[1]])  # no slot
    with pytest.raises(RuntimeError):
        b.capture()
    with pytest.raises(RuntimeError):
        b.generate([p[1]], 2)
    with pytest.raises(ValueError):
        b.step(tok[:2])
    assert state[0] == b.lengths and state[1] == len(b.allocator)
    assert torch.equal(state[2], b._table) and torch.equal(state[3], b._lens)
    for s in list(b.active()):
        b.release(s)
    assert len(b.allocator) == 12 and int(b._lens.sum()) == 0
    few = _batch(d, num_pages=2)
    with pytest.raises(RuntimeError):
        few.add([p[0], p[1]])  # three pages
    slots, _ = few.add([torch.zeros(32, dtype=torch.long)])
    with pytest.raises(RuntimeError):
        few.step(tok)  # a third page
    assert few.lengths[slots[0]] == 32
    full = _batch(d, max_seq=20)
    full.add([p[0]])
    with pytest.raises(ValueError):
        full.step(tok)


@gpu
def test_generate_where_the_room_ends():
    """max_seq and the pages: refused as a whole beforehand without eos; with one
    that is not drawn each sequence ends where it finds no room, and the others
    go on with its pages; what was drawn is what a larger cache gives."""
    _, d = _parts()
    prompts = [torch.tensor(p) for p in PROMPTS]  # of 20, 7, 1 and 16 tokens
    kw = dict(temperature=0.0)
    big = _batch(d, num_pages=16)
    want = big.generate(prompts, 30, **kw)
    never = next(t for t in range(CFG["vocab_size"]) if all(t not in r for r in want))
    calls = []
    short = _batch(d, max_seq=24)
    short.add = lambda p, add=short.add: calls.append(len(p)) or add(p)
    with pytest.raises(ValueError):
        short.generate(prompts, 6, **kw)
    assert not calls and short.generate(prompts, 5, **kw) == [r[:5] for r in want]
    # 24 positions hold a prompt of n and 24 - n tokens, and one more is drawn
    assert short.generate(prompts, 30, eos=never, **kw) == [r[: min(30, 25 - len(p))] for r, p in zip(want, PROMPTS)]
    assert len(short.allocator) == 12 and not short.active()
    few = _batch(d, num_pages=6)
    with pytest.raises(RuntimeError):
        few.generate(prompts, 30, **kw)
    assert not few.active() and len(few.allocator) == 6
    # five pages hold the prompts; the fourth needs a second page at once and takes the last; the second, at 16, finds
    # none and ends with 16 - 7 + 1 tokens, and its page serves the first, at 32
    got = few.generate(prompts, 30, eos=never, **kw)
    lens = [len(r) for r in got]
    assert lens[1] == 10 and max(lens) == 30 and all(r == w[: len(r)] for r, w in zip(got, want))
    assert len(few.allocator) == 6 and not few.active()
    stop = want[1][3]
    cut = few.generate(prompts[1:2], 30, eos=stop, **kw)
    assert cut == [want[1][: want[1].index(stop) + 1]]


@gpu
def test_refused_steps_change_nothing():
    """Ids on the host, of no integer type or no ids at all: lengths, pages and
    the device's lengths stay; the next step gives what it gives without them."""
    _, d = _parts()
    tok = torch.tensor([11, 12, 13, 14], device="cuda")
    out = []
    for bad in ([], [tok.cpu(), tok.float(), tok.half(), tok[:2], tok[None], tok.cpu().int()]):
        b = _batch(d)
        b.add([torch.tensor(PROMPTS[3]), torch.tensor(PROMPTS[1])])  # 16 tokens: the next one needs a page
        for t in bad:
            with pytest.raises(ValueError):
                b.step(t)
            assert b.lengths == [16, 7, 0, 0] and len(b.allocator) == 12 - 2 and b._lens.tolist() == [16, 7, 0, 0]
        out.append(b.step(tok.int() if bad else tok)[:2].clone())
    assert torch.equal(*out)


def _give_up(monkeypatch):
    """prompt_attention's kernel gives up wherever it has to wait."""
    from polarflash_b200 import _lib

    L = _lib.load()
    monkeypatch.setattr(L, "pf_prompt_attention", lambda *a: L.pf_prompt_selftest(*a[:-1], 0, a[-1]))


@gpu
def test_prompts_whose_attention_gave_up_are_taken_back(monkeypatch):
    _, d = _parts()
    b = _batch(d)
    want = b.add([torch.tensor(PROMPTS[0])])[1]
    with monkeypatch.context() as m:
        _give_up(m)
        with pytest.raises(RuntimeError, match="timed out"):
            b.add([torch.tensor(p) for p in PROMPTS[1:3]])
    assert b.active() == [0] and len(b.allocator) == 12 - 2 and b._lens.tolist() == [20, 0, 0, 0]
    slots, got = b.add([torch.tensor(PROMPTS[0])])  # nothing is left to report
    assert slots == [1] and torch.equal(got, want)


@gpu
def test_generate():
    """Greedy tokens are the argmax of the steps' logits, batch and single
    decoder alike up to near ties; the same generator state gives the same
    draws; eos ends a sequence; replays equal eager steps."""
    w, d = _parts()
    b, bg = _batch(d), _batch(d)
    bg.capture()
    prompts = [torch.tensor(p) for p in PROMPTS]
    greedy = b.generate(prompts, 6, temperature=0.0)
    assert [len(r) for r in greedy] == [6] * 4 and len(b.allocator) == 12
    assert bg.generate(prompts, 6, temperature=0.0) == greedy
    slots, logits = b.add(prompts)
    tok = torch.zeros(4, dtype=torch.long, device="cuda")
    for t in range(6):
        tok[:] = logits.argmax(-1)
        assert tok.tolist() == [r[t] for r in greedy]
        logits = b.step(tok)
    for s in slots:
        b.release(s)
    kw = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    gen = lambda s: torch.Generator(device="cuda").manual_seed(s)  # noqa: E731
    a1, a2, a3 = (b.generate(prompts, 8, generator=gen(s), **kw) for s in (1, 1, 2))
    assert a1 == a2 and a1 != a3
    eos = a1[0][2]
    cut = b.generate(prompts, 8, generator=gen(1), eos=eos, **kw)
    assert cut[0] == a1[0][: a1[0].index(eos) + 1] and len(b.allocator) == 12
    assert b.generate(prompts, 0) == [[]] * 4
    # one sequence
    d.capture()
    d.length = 0
    single = d.generate(torch.tensor(PROMPTS[0], device="cuda"), 5, temperature=0.0)
    assert d.length == len(PROMPTS[0]) + 4
    caches = [{} for _ in range(CFG["num_hidden_layers"])]
    ref, ids = [], PROMPTS[0]
    for _ in range(5):
        ref.append(int(dm.reference_forward(w, ids, caches)[-1].argmax()))
        ids = [ref[-1]]
    assert single == ref
    d.length = 0
    one = d.generate(torch.tensor(PROMPTS[0], device="cuda"), 9, temperature=0.0, eos=ref[1])
    assert one == ref[: ref.index(ref[1]) + 1]


@gpu
@pytest.mark.parametrize("dt,tol", [(torch.float16, 1e-2), (torch.bfloat16, 8e-2)])
@pytest.mark.parametrize("kv", ["fp32", "int8"])
def test_prompt_dtype_of_the_single_decoder(dt, tol, kv):
    """A prompt in two parts (the second over the first's cache) with 16-bit
    attention against the fp32 default."""
    from test_decode_step import _decoder

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    w = dm.build()
    a, b = _decoder(w, kv_mode=kv), _decoder(w, kv_mode=kv)
    b.prompt_dtype = dt
    ids = torch.tensor(dm.PROMPT, device="cuda")
    for part in (ids[:13], ids[13:], ids[:1]):
        assert _rel(b.forward(part), a.forward(part)) < tol
    from polarflash_b200.decode import PFlashDecoder

    with pytest.raises(ValueError):
        PFlashDecoder(CFG, a.layers, a.embed, a.final_norm, a.lm_head, 8, prompt_dtype=torch.float32)


@gpu
def test_prompt_dtype_that_gave_up_raises(monkeypatch):
    from test_decode_step import _decoder

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    d = _decoder(dm.build())
    d.prompt_dtype = torch.bfloat16
    ids = torch.tensor(dm.PROMPT, device="cuda")
    want = d.forward(ids[:9]).clone()
    with monkeypatch.context() as m:
        _give_up(m)
        for call in (lambda: d.forward(ids[9:]), lambda: d.generate(ids[9:], 3)):
            with pytest.raises(RuntimeError, match="timed out"):
                call()
            assert d.length == 9
    d.length = 0
    assert torch.equal(d.forward(ids[:9]), want)
