"""GPU: a model on the 4-bit K/V cache (DecodeEngine(kv_bits=4)) against a plain model in single precision whose keys and values are the cache's."""
import subprocess
import sys

import pytest
import torch

from flint_b200 import _lib, packing
from flint_b200.config import ModelArgs
from flint_b200.draft import seeded_draft
from flint_b200.engine import DecodeEngine
from flint_b200.generate import generate, generate_tree
from flint_b200.kv4 import KvCache4
from flint_b200.model import Transformer
from flint_b200.tree import static_tree, tree_mask
from oracle import oracle as O
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"

CONFIGS = {
    "tiny": ModelArgs.from_name("tiny"),                                        # heads of 64
    "tiny-window": ModelArgs.from_name("tiny-window"),                          # of 80
    "8b-shape": ModelArgs(block_size=512, vocab_size=1000, n_layer=2, n_head=32, n_local_heads=8, dim=4096, intermediate_size=14336, rope_base=500000),   # of 128
}


class Plain:
    """The passes' arithmetic with bf16 roundings where they round, one layer after the other; K and V rows as the 4-bit cache holds them."""

    def __init__(self, cfg, packed):
        self.cfg, self.embed = cfg, packed["embed"].to(DEV).float()
        w = lambda n, i: torch.from_numpy(O.c_dequant(packed[n + "_q"][i] if i is not None else packed[n + "_q"],  # noqa: E731
                                                      packed[n + "_s"][i] if i is not None else packed[n + "_s"],
                                                      None if n + "_z" not in packed else packed[n + "_z"][i] if i is not None else packed[n + "_z"])).to(DEV)
        self.layers = [{n: w(n, i) for n in ("qkv", "o", "gu", "d")} for i in range(cfg.n_layer)]
        self.lm = w("lm", None)
        self.n1, self.n2, self.nf = (packed[n].to(DEV).float() for n in ("n1", "n2", "nf"))
        self.K = [torch.zeros(0, cfg.n_local_heads, cfg.head_dim, device=DEV) for _ in range(cfg.n_layer)]
        self.V = [k.clone() for k in self.K]

    def step(self, tokens, pos, depth=None, amask=None):
        cfg, b = self.cfg, lambda x: x.bfloat16().float()  # noqa: E731
        n, nh, nkv, hd, F = len(tokens), cfg.n_head, cfg.n_local_heads, cfg.head_dim, cfg.ffn_padded
        norm = lambda x, w: b(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.norm_eps) * w)  # noqa: E731
        where = pos + (torch.arange(n, device=DEV) if depth is None else depth)
        h = b(self.embed[tokens] * cfg.embedding_multiplier)
        for i, w in enumerate(self.layers):
            q, k, v = (b(norm(h, self.n1[i]) @ w["qkv"].T)).view(n, nh + 2 * nkv, hd).split([nh, nkv, nkv], 1)
            q = ref.rotated(q.bfloat16(), where, cfg.rope_base).bfloat16()
            k, v = ref.values(ref.rotated(k.bfloat16(), where, cfg.rope_base).float()), ref.values(v)
            self.K[i], self.V[i] = torch.cat([self.K[i][:pos], k]), torch.cat([self.V[i][:pos], v])
            a = b(ref.attention(q, self.K[i], self.V[i], pos, cfg.attn_scale, amask).float()).reshape(n, -1)
            h = b(h + a @ w["o"].T * cfg.residual_multiplier)
            g, u = b(norm(h, self.n2[i]) @ w["gu"].T).split([F, F], -1)
            h = b(h + b(torch.nn.functional.silu(g) * u) @ w["d"].T * cfg.residual_multiplier)
        f = norm(h, self.nf)
        return f @ self.lm.T / cfg.logits_scaling, f, h

    def move(self, src, dst):
        for x in self.K + self.V:
            for a, c in zip(src, dst):
                x[c] = x[a].clone()


def near(got, want, most=0.03):
    """Both sides round to bf16 six times a layer (half a step: 2^-8 of a value, 0.0023 of the norm); they sum in different orders, so some of these roundings go
    the other way, and of the nibbles whose numbers differ by a step of bf16 about one in a hundred. All roundings of four layers apart would be
    0.0023 sqrt(24) = 0.011 of the norm, the nibbles about as much."""
    rel = float((got.float() - want).norm() / want.norm())
    assert rel <= most, rel


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("asym", [False, True])
def test_prompt_tree_compaction_and_decoding(name, asym):
    cfg = CONFIGS[name]
    packed = packing.synth_packed(cfg, 1, device="cpu", asym=asym)
    model = Plain(cfg, packed)
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, cfg.vocab_size, (90,), generator=g).to(DEV)
    # a cache whose pages lie in any order, with pages of somebody else's between them
    table = torch.tensor([[5, 1, 7, 2]], dtype=torch.int32, device=DEV)
    cache = KvCache4(cfg.n_layer, 9, cfg.n_local_heads, cfg.head_dim, table, rope_base=cfg.rope_base)
    cache.pool.fill_(0xFF)
    eng = DecodeEngine(cfg, {k: v.to(DEV) for k, v in packed.items()}, kv_bits=4, cache=cache)
    assert eng.max_seq == 256 and eng.cache is cache and eng.kc is None
    logits, feat = eng.prefill(prompt[:85], 0)                                   # more than 64 tokens, then few
    want, wf, _ = model.step(prompt[:85], 0)
    near(logits, want)
    near(feat, wf)
    logits, _ = eng.verify(prompt[85:], 85)
    near(logits, model.step(prompt[85:], 85)[0])
    pos = 90
    parent, depth = static_tree(9)
    nodes = torch.randint(0, cfg.vocab_size, (9,), generator=g).to(DEV)
    amask = torch.from_numpy(tree_mask(parent)).to(DEV)
    depth = torch.tensor(depth, dtype=torch.int32, device=DEV)
    logits, _ = eng.verify(nodes, pos, depth, amask)
    near(logits, model.step(nodes, pos, depth, amask)[0])
    path = [0, 2, 6]
    eng.kv_compact(torch.tensor([3, 0] + path + [0] * 6, dtype=torch.int32, device=DEV), pos)
    model.move([pos + p for p in path], [pos + i for i in range(3)])
    eng.kv_move([3, 4], [4, 3])
    model.move([3, 4], [4, 3])
    pos += 3
    tok = torch.tensor([11], dtype=torch.int32, device=DEV)
    for i in range(5):
        want, _, h = model.step(tok.long(), pos + i)
        if i == 0:
            got = eng.decode(int(tok), pos)
        elif i == 1:
            got = torch.empty(cfg.vocab_size, dtype=torch.float32, device=DEV)
            eng.decode_chained(tok, pos + i, eng.next_token, got)
        elif i == 2:                                                             # the caller's embedding, which becomes the final residual
            x = (packed["embed"][int(tok)].to(DEV).float() * cfg.embedding_multiplier).bfloat16()
            got = eng.decode_h(x, pos + i)
            near(x.view(1, -1), h)
        elif i == 3:
            eng.decode_chained(tok, pos + i, eng.next_token)                     # no logits asked for
            got = None
        else:
            got = eng.decode(int(tok), pos + i)
        if got is not None:
            near(got.view(1, -1), want)
            assert int(eng.next_token) == int(got.argmax())
        tok = eng.next_token.clone()
    eng.check()
    # Rows on both sides are the same numbers but for roundings. Behind the first layer the numbers differ by up to r = 0.03 of their norm; a nibble's step is about
    # 0.35 of it (15 steps from the smallest to the largest of 64 to 128 normal numbers), so that a share 0.8 r / 0.35 of the nibbles goes one step the other way:
    # sqrt(0.8 r / 0.35) 0.35 = 0.09 of the norm, and r itself
    for i in range(cfg.n_layer):
        K, V = cache.read(i, pos + 5, 0)
        near(K, model.K[i][:pos + 5], 0.12 if i else 0.03)
        near(V, model.V[i][:pos + 5], 0.12 if i else 0.03)
    others = [p for p in range(9) if p not in (5, 1, 7, 2)]
    assert (cache.pool[:, others] == 0xFF).all()
    eng.close()


def test_generate_on_four_bits():
    """generate() is the same plumbing on either cache: the prompt pass, then the chained decode loop, bit for bit; a captured step among them."""
    model = Transformer.from_name("tiny", kv_bits=4).load_synthetic(seed=0)
    prompt = torch.randint(0, 4096, (70,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    seq, _ = generate(model, prompt, 20)
    eng = DecodeEngine(model.config, model.packed, max_seq=96, kv_bits=4)
    assert eng.max_seq == 128
    out = torch.zeros(20, dtype=torch.int32, device=DEV)
    lg, _ = eng.prefill(prompt, 0)
    out[0] = lg[-1].argmax()
    for i in range(10):
        eng.decode_chained(out[i:i + 1], 70 + i, out[i + 1:i + 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for i in range(10, 19):
                eng.decode_chained(out[i:i + 1], 70 + i, out[i + 1:i + 2])
        graph.replay()
    torch.cuda.synchronize()
    eng.check()
    assert torch.equal(out, seq[70:])
    # speculation accepts what greedy decoding would have said: near-ties apart, the same tokens
    draft = seeded_draft(512, 8, 1376, seed=1)
    tree, st = generate_tree(model, prompt, 20, draft, beam=2, depth=3)
    chain, _ = generate(model, prompt, 20, draft_model=draft, speculate_k=3)
    check = DecodeEngine(model.config, model.packed, max_seq=96, kv_bits=4)
    for s in (tree, chain):
        toks = s.tolist()
        for pos in range(len(toks) - 1):
            lg = check.decode(toks[pos], pos)
            if pos >= 69:
                assert float(lg.max() - lg[toks[pos + 1]]) <= 0.05
    check.check()


def test_the_cache_bound_last_is_used():
    cfg = ModelArgs.from_name("tiny")
    packed = packing.synth_packed(cfg, 0, device=DEV)
    eng = DecodeEngine(cfg, packed, max_seq=64)
    toks = list(range(5, 15))
    first = [eng.decode(t, i).clone() for i, t in enumerate(toks)]
    kc, vc = eng.kc, eng.vc
    four = KvCache4(cfg.n_layer, 1, 2, 64, torch.zeros(1, 1, dtype=torch.int32, device=DEV), rope_base=cfg.rope_base)
    keep = kc.clone()
    eng.bind_kv4(four)
    lg = [eng.decode(t, i).clone() for i, t in enumerate(toks)]
    assert torch.equal(kc, keep) and four.pool.any() and not torch.equal(lg[-1], first[-1])
    with pytest.raises(_lib.FlintError) as e:
        eng.decode(1, 64)
    assert e.value.code == _lib.FB_ERR_RANGE
    eng.bind_kv(kc, vc)
    for i, t in enumerate(toks):
        assert torch.equal(eng.decode(t, i), first[i])
    eng.check()


def test_refused_engines():
    cfg = ModelArgs.from_name("tiny")
    packed = packing.synth_packed(cfg, 0, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    kc = torch.zeros(4, 64, 2, 64, dtype=torch.bfloat16, device=DEV)
    good = lambda **kw: KvCache4(**{**dict(n_layer=4, n_pages=2, n_kv=2, head_dim=64, table=table, rope_base=1e4), **kw})  # noqa: E731
    for kw in (dict(kv_bits=8), dict(kv_bits=4, kc=kc, vc=kc), dict(kv_bits=16, cache=good()), dict(kv_bits=4, cache=good(n_layer=3)), dict(kv_bits=4, cache=good(n_kv=1)),
               dict(kv_bits=4, cache=good(head_dim=80)), dict(kv_bits=4, cache=good(rope_base=None)), dict(kv_bits=4, cache=good(table=table.repeat(2, 1)))):
        with pytest.raises(ValueError):
            DecodeEngine(cfg, packed, **kw)
    with pytest.raises(ValueError):
        Transformer(cfg, kv_bits=5)
    eng = DecodeEngine(cfg, packed, kv_bits=4, cache=good())
    for call in (lambda: eng.decode(5, 128), lambda: eng.decode(5, -1), lambda: eng.decode(4096, 0), lambda: eng.verify([1, 2], 127), lambda: eng.prefill([1] * 129, 0),
                 lambda: eng.kv_move([0], [128]), lambda: eng.kv_compact(torch.zeros(3, dtype=torch.int32, device=DEV), 128)):
        with pytest.raises(_lib.FlintError) as e:
            call()
        assert e.value.code == _lib.FB_ERR_RANGE
    eng.check()
    table[0, 1] = 9                                                              # a page that is none: reported by the engine's status
    eng.decode(5, 64)
    with pytest.raises(_lib.FlintError) as e:
        eng.check()
    assert e.value.code == _lib.FB_ERR_RANGE


def test_chat_on_four_bits():
    run = subprocess.run([sys.executable, "chat.py", "--config", "tiny", "--maxseq", "256", "--max-new", "8", "--kv-bits", "4"], input="5 17 99\n12 13\n", capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-500:]
    assert run.stdout.count("8 tokens") == 2


@pytest.mark.parametrize("name,M,pos", [("tiny", 1, 0), ("tiny", 3, 600), ("tiny", 40, 0), ("tiny", 300, 0), ("tiny", 16, 600), ("llama-8b-class", 1, 3000),
                                        ("llama-8b-class", 26, 1500), ("llama-8b-class", 61, 700), ("llama-8b-class", 200, 700)])
def test_passes_that_give_up_leave_nothing_behind(name, M, pos):
    """A wait limit of 0: every launch ends, after what it has in flight (that wait has its own limit), the status says time-out or, if every wait happened to be
    satisfied, nothing, and the next clean pass gives the bits of the first."""
    cfg = ModelArgs.from_name(name)
    if name != "tiny":
        cfg.n_layer, cfg.vocab_size = 1, 512
    eng = DecodeEngine(cfg, packing.synth_packed(cfg, 0, device=DEV), max_seq=pos + 512, kv_bits=4)
    g = torch.Generator(device=DEV).manual_seed(pos)
    for layer in range(cfg.n_layer if pos else 0):
        k, v = (torch.randn(pos, cfg.n_local_heads, cfg.head_dim, generator=g, device=DEV).bfloat16() for _ in range(2))
        eng.cache.append(layer, k, v, 0)
    toks = torch.randint(0, cfg.vocab_size, (M,), generator=torch.Generator().manual_seed(M), dtype=torch.int32).to(DEV)
    run = (lambda: eng.decode(17, pos).clone()) if M == 1 else (lambda: (eng.verify if M <= 64 else eng.prefill)(toks, pos)[0])
    want = run()
    eng.check()
    for _ in range(8):
        eng.set_option(0, 0)
        run()
        assert eng.status()["code"] in (_lib.FB_OK, _lib.FB_ERR_TIMEOUT)
        eng.set_option(0, 4000000)
        again = run()
        eng.check()
        assert torch.equal(want, again)
