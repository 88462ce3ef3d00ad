"""The attention layer and the engine over a packed cache: portions, decoded tokens, mixed and captured steps."""
import pytest
import torch

import plain_llama as P
import plain_packed as plain
import tiny_configs
import trace_tools as tt
from mixer_tools import make_kit

pytestmark = pytest.mark.gpu

F64 = torch.float64


@pytest.fixture(scope="module")
def kit(cuda_device):
    return make_kit()


LAYERS = [dict(nh=8, nkv=2, d=64, page=16), dict(nh=4, nkv=1, d=128, page=16, window=40), dict(nh=6, nkv=3, d=32, page=8, rot=16, interleaved=True),
          dict(nh=4, nkv=2, d=128, page=32, window=50, sink=True, distance_bias=True, temperature=(0.1, 16)), dict(nh=3, nkv=1, d=64, page=16, softcap=8.0)]


def build(kit, dtype, layer, bits):
    c = dict(layer)
    nh, nkv, d, page = c.pop("nh"), c.pop("nkv"), c.pop("d"), c.pop("page")
    rot, inter = c.pop("rot", d), c.pop("interleaved", False)
    ctx = kit.parts.BuildContext(dtype, "cuda", max_tokens=512, max_seqs=8, page_size=page, cache_bits=bits)
    pos = kit.parts.PartSpec("none") if c.get("distance_bias") else \
        kit.parts.PartSpec("rope", dict(head_dim=d, rotary_dim=rot, theta=5000.0, interleaved=inter))
    mixer = kit.parts.build_mixer(kit.parts.PartSpec("attention", dict(hidden_size=96, num_heads=nh, num_kv_heads=nkv, head_dim=d, position=pos, **c)), ctx)
    g = torch.Generator().manual_seed(4)
    w = {n: (torch.randn(s.shape, generator=g) * (0.2 if len(s.shape) == 2 else 1.0)).to(dtype) for n, s in mixer.weights().items()}
    mixer.load(lambda n: w[n].cuda())
    return mixer, w


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", range(len(LAYERS)))
def test_layer(kit, which, dtype, bits):
    """Two sequences in portions, mixed steps and single tokens.  What the pages hold is checked against the formula (within
    half a step, and the rounding of the projections), and the output against attention over what they hold."""
    layer = LAYERS[which]
    nh, nkv, d, page = (layer[k] for k in ("nh", "nkv", "d", "page"))
    mixer, w = build(kit, dtype, layer, bits)
    need = mixer.cache_need()
    assert need.bits == bits
    cm = kit.CacheManager([need], page, 40, 4, dtype=dtype, device="cuda")
    bb = kit.BatchBuilder(cm, "cuda", query_tiles=mixer.query_tiles())
    g = torch.Generator().manual_seed(which)
    x = {s: torch.randn(90, 96, generator=g).to(dtype) for s in "ab"}
    steps = [dict(a=20), dict(a=1, b=33), dict(a=1, b=1), dict(a=30, b=1), dict(b=2), dict(a=1, b=17), dict(a=1, b=1)]
    at, outs = dict(a=0, b=0), dict(a=[], b=[])
    for s in "ab":
        cm.admit(s)
    for step in steps:
        batch = bb.build([kit.StepEntry(s, [0] * n, []) for s, n in step.items()])
        rows = torch.cat([x[s][at[s]:at[s] + n] for s, n in step.items()]).cuda()
        y = mixer.forward(rows, batch, cm.layer_cache(0)).cpu().double()
        for s, n in step.items():
            outs[s].append(y[:n])
            y = y[n:]
            at[s] += n
    inv = 5000.0 ** (-torch.arange(0, layer.get("rot", d), 2, dtype=F64) / layer.get("rot", d))
    kv = cm.layer_cache(0)[0]
    pages = kv.pages.cpu()
    exact = dtype == torch.float32
    o = {k: layer[k] for k in ("window", "softcap", "temperature") if k in layer}
    if layer.get("sink"):
        o["sink"] = w["sink"].float()
    if layer.get("distance_bias"):
        o["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)])
    for s in "ab":
        n = at[s]
        xd = x[s][:n].double()
        q, k, v = ((xd @ w[f"{c}_proj.weight"].double().T) for c in "qkv")
        if not exact:                      # the projections round once; the rotation of what they leave is float32
            q, k, v = (t.to(dtype).double() for t in (q, k, v))
        q, k, v = q.view(n, nh, d), k.view(n, nkv, d), v.view(n, nkv, d)
        if not layer.get("distance_bias"):
            for i in range(n):
                q[i] = plain.rotate(q[i], float(i), inv, layer.get("interleaved", False))
                k[i] = plain.rotate(k[i], float(i), inv, layer.get("interleaved", False))
        table = cm.block_table(s, 0)
        held = torch.zeros(2, n, nkv, d, dtype=F64)
        for i in range(n):
            if table[i // page] < 0:       # given back behind the window
                continue
            for h in range(nkv):
                a, b = plain.get(pages, table[i // page] * page + i % page, h, d, bits, page)
                held[0, i, h], held[1, i, h] = a, b
                for y, t in ((a, k[i, h]), (b, v[i, h])):
                    _, scale, _ = plain.quantise(t, bits)
                    # half a step, what a product in another order changes of it (bfloat16: one more rounding), and the scale's own step
                    slack = (2.0 ** -18 if exact else 2.0 ** -7) * t.abs().max() + scale.max() * 2.0 ** -6
                    assert ((y - t).abs() <= 0.5 * scale.max() + slack).all()
        got = torch.cat(outs[s])
        first = 0 if not layer.get("window") else max(0, n - layer["window"])          # earlier rows saw pages that are gone by now
        ref = plain.attend(q[first:], held[0], held[1], n, d ** -0.5, **o)
        lo = 0
        for i in range(first, n):          # rows whose whole window is still held
            if layer.get("window") and any(table[j // page] < 0 for j in range(max(0, i - layer["window"] + 1), i + 1)):
                lo = i - first + 1
        want = ref[lo:].reshape(n - first - lo, nh * d) @ w["o_proj.weight"].double().T
        err = float((got[first + lo:] - want).abs().max() / want.abs().max())
        assert err <= (2e-5 if exact else 3e-2), err


def test_captured_steps_follow_contexts_and_streams(kit):
    """A step captured once is replayed with other contexts, slots and pages; two captured steps and an eager one on other
    streams do not disturb one another."""
    from gollmgo_b200.cache import PackedKV
    nh, nkv, d, page, n = 8, 2, 128, 16, 5
    kv = PackedKV.empty(64, nkv, d, page, 4)
    g = torch.Generator().manual_seed(0)
    width = 12
    tables = torch.randperm(64, generator=g)[:n * width].view(n, width).to(torch.int32).cuda()
    rows = torch.randn(64 * page, (nh + 2 * nkv) * d, generator=g).to(torch.bfloat16).cuda()
    kv.write(rows, None, torch.arange(64 * page, dtype=torch.int32).cuda(), nh)
    q = torch.randn(n, nh, d, generator=g).to(torch.bfloat16).cuda()
    contexts = [torch.tensor(c, dtype=torch.int32).cuda() for c in ([3, 17, 64, 100, 192], [190, 1, 0, 33, 32], [16, 16, 16, 16, 16])]
    want = [kv.decode(q, tables, c, 192, 0.1).clone() for c in contexts]
    live = [contexts[0].clone(), contexts[1].clone()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in live:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            kv.decode(q, tables, c, 192, 0.1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kv.decode(q, tables, c, 192, 0.1))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b in ((0, 1), (2, 0), (1, 2)):
        live[0].copy_(contexts[a])
        live[1].copy_(contexts[b])
        torch.cuda.synchronize()
        for _ in range(10):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            eager = kv.decode(q, tables, contexts[2], 192, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b]) and torch.equal(eager, want[2])


def test_write_read_and_portions_are_captured_too(kit):
    from gollmgo_b200.cache import PackedKV
    nh, nkv, d, page = 4, 2, 64, 16
    kv = PackedKV.empty(16, nkv, d, page, 8)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(60, (nh + 2 * nkv) * d, generator=g).to(torch.bfloat16).cuda()
    tables = torch.tensor([[3, 1, 9], [0, 7, -1]], dtype=torch.int32).cuda()
    pos = torch.cat([torch.arange(40), torch.arange(20)]).to(torch.int32).cuda()
    seq = torch.tensor([0] * 40 + [1] * 20).cuda()
    slots = (tables[seq, pos.long() // page] * page + pos % page).to(torch.int32)
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    cu, ctx, first = dev([0, 40, 60]), dev([40, 20]), dev([0, 3])
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=F64, device="cuda") / d)

    def run():
        q = kv.write(rows, pos, slots, nh, inv)
        return q, *kv.read(tables, ctx, first, 5), kv.prefill(q, tables, cu, ctx, [40, 20], [40, 20], 0.125)
    want = [t.clone() for t in run()]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    kv.pages.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- the engine
@pytest.fixture(scope="module")
def models(tmp_path_factory, cuda_device):
    tmp = str(tmp_path_factory.mktemp("models"))
    out = {}
    for name in ("tiny_a", "tiny_d", "tiny_e"):
        cfg, page, std, jitter = tiny_configs.get(name)
        folder = tt.model_folder(tmp, name, cfg, seed=21, std=std, jitter=jitter, dtype="float32")
        out[name] = (folder, cfg, page, tt.load_weights(folder))
    return out


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("name", ["tiny_a", "tiny_d", "tiny_e"])
def test_logits_of_a_quantised_plain_model(models, name, bits, monkeypatch):
    """float32 steps (a prompt in portions, then single tokens) against the plain model whose attention sees keys and values as
    they read once stored.  A key that float32 products leave on the other side of a border between two codes changes its value by a step, one of
    n tokens and d channels: the tolerance allows a few of those (a step is 1/15 or 1/255 of a group's range)."""
    from gollmgo_b200.config import EngineConfig
    from gollmgo_b200.engine.batch import StepEntry
    from gollmgo_b200.engine.runner import load_runner
    folder, cfg, page, w = models[name]
    old = P.attention
    monkeypatch.setattr(P, "attention", lambda q, k, v, window=None: old(q, plain.through(k.double().cpu(), bits).to(k.device),
                                                                          plain.through(v.double().cpu(), bits).to(v.device), window))
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(0, cfg["vocab_size"], (75,), generator=g).tolist()
    want = P.forward(w, cfg, tokens)
    runner = load_runner(folder, EngineConfig(dtype="float32", block_size=page, num_blocks=32, max_batch_size=4, max_token_budget=64, cache_bits=bits,
                                              cuda_graphs=True, capture_at_start=False))
    runner.cache.poison_freed = True
    at, rows = 0, []
    for n in [30, 17, 1, 1, 20] + [1] * 6:
        rows.append(runner.step([StepEntry("r", tokens[at:at + n], list(range(n)))]).cpu().double().clone())
        at += n
    got = torch.cat(rows)
    err = float((got - want.cpu().double()).abs().max() / want.abs().max())
    assert err <= (2e-2 if bits == 4 else 2e-3), err


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("name", ["tiny_a", "tiny_d", "tiny_e"])
def test_engine_runs_and_gives_its_pages_back(models, name, bits, dtype):
    """Batches with chunked prompts, captured decode steps and a pool so small that requests are preempted; the same again."""
    from gollmgo_b200 import Engine, SamplingParams
    folder, cfg, page, w = models[name]
    reqs = list(tt.random_requests(cfg["vocab_size"], [7, 33, 1, 60, 21], seed=1).values())
    outs = []
    for _ in range(2):
        eng = Engine(folder, dtype=dtype, block_size=page, num_blocks=3 + 160 // page, max_batch_size=4, max_token_budget=48, prefill_chunk_size=24,
                     cache_bits=bits)
        eng.runner.cache.poison_freed = True
        res = eng.generate(reqs, SamplingParams(max_tokens=12, ignore_eos=True))
        assert all(len(o.token_ids) == 12 and o.finish_reason == "length" for o in res)
        eng.runner.cache.audit()
        assert eng.runner.cache.free_pages() == 3 + 160 // page
        eng.runner.check_kernels()
        outs.append([o.token_ids for o in res])
    assert outs[0] == outs[1]


def test_memory_holds_more_tokens(models):
    from gollmgo_b200.config import EngineConfig
    from gollmgo_b200.cache import CacheManager
    from gollmgo_b200.engine.runner import load_runner
    folder, cfg, page, w = models["tiny_e"]
    got = {}
    for bits in (None, 8, 4):
        r = load_runner(folder, EngineConfig(dtype="bfloat16", block_size=page, max_memory_fraction=0.02, max_batch_size=4, max_token_budget=64,
                                             max_model_len=512, cache_bits=bits, cuda_graphs=False))
        got[bits] = r.num_pages
        del r
        torch.cuda.empty_cache()
    assert got[8] > 1.8 * got[None] and got[4] > 3.4 * got[None]
