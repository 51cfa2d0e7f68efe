"""The decode step's options through the decoder: 4-bit weights, sparse attention, logit controls,
each alone and all of them together, with and without CUDA graphs."""

import copy

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.config import Qwen3Config, Sampling
from helios_b200.controls import LogitControls, TokenHistory, control_rows
from helios_b200.decode import Decoder, sample_rows
from helios_b200.model import Qwen3Model
from helios_b200.paged_cache import KVPagePool, PagedKVCache, SparseAttention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
SHAPE = dict(vocab_size=4096, context_length=4096, hidden_size=512, n_heads=8, n_layers=2, hidden_dim=1024,
             head_dim=128, n_kv_heads=2, rope_base=1e6, rms_norm_eps=1e-6, dtype=torch.bfloat16)
GREEDY = Sampling(max_new_tokens=1, temperature=0, top_p=1)


def _model(seed=0):
    torch.manual_seed(seed)
    return Qwen3Model(Qwen3Config(**SHAPE)).to(DEV).eval()


def _decoder(model, pages=48, **kw):
    decoder = Decoder(model)
    decoder.page_pool = KVPagePool(model.config, pages, device=DEV)
    for name, value in kw.items():
        setattr(decoder, name, value)
    return decoder


def _prompts(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lengths]


def _close(a, b):
    # bf16 roundings in another order (see test_gpu_graphs): 2% of the row's largest logit.
    scale = b.float().abs().amax(dim=-1, keepdim=True).clamp(min=1.0)
    assert ((a.float() - b.float()).abs() <= 2e-2 * scale).all()


def _decode(decoder, prompts, steps, greedy=True):
    """Logits of the prompts' last positions and of ``steps`` greedy decode ticks."""
    caches = [PagedKVCache(decoder.page_pool, len(p) + steps + 1) for p in prompts]
    logits = [decoder.packed_caches(caches, prompts).clone()]
    for _ in range(steps):
        logits.append(decoder.decode_caches(caches, logits[-1].argmax(-1)).clone())
    for cache in caches:
        cache.close()
    return logits


@pytest.mark.parametrize("group", [32, 128])
def test_quantized_model_is_the_model_of_its_weights(group):
    """Weights that 4 bits hold exactly: k / 8 with |k| <= 7 in every group, so the scale is 1/8 (a power
    of two) and the 4-bit model computes with the same weights as the bf16 one."""
    model = _model()
    g = torch.Generator(device=DEV).manual_seed(5)
    with torch.no_grad():
        for block in model.blocks:
            for linear in (block.attention.query, block.attention.key, block.attention.value, block.attention.output,
                           block.feed_forward.gate, block.feed_forward.up, block.feed_forward.down):
                w = torch.randint(-7, 8, linear.weight.shape, generator=g, device=DEV)
                w[:, ::group] = 7
                linear.weight.copy_((w / 8).to(torch.bfloat16) / 16)
    twin = copy.deepcopy(model)
    model.quantize_weights(group)
    assert model.blocks[0].feed_forward.gate.weight.numel() == 0
    with pytest.raises(RuntimeError, match="already"):
        model.quantize_weights(group)
    prompts = _prompts((3, 40, 200))
    for a, b in zip(_decode(_decoder(model), prompts, 6), _decode(_decoder(twin), prompts, 6)):
        _close(a, b)
    with pytest.raises(RuntimeError):  # the full-precision weights have no place to go
        model.load_state_dict(twin.state_dict())
    assert _native.device_status() == 0


def test_quantizing_drops_captured_ticks():
    model = _model()
    model.enable_cuda_graphs()
    decoder = _decoder(model)
    prompts = _prompts((5, 30))
    _decode(decoder, prompts, 4)
    model.quantize_weights(64, symmetric=False)
    graphed = _decode(decoder, prompts, 5)
    assert model._graphs.replays > 0
    model._graphs = None
    for a, b in zip(graphed, _decode(_decoder(model), prompts, 5)):
        _close(a, b)


def test_sparse_attention_over_every_block_is_dense():
    model = _model()
    prompts = _prompts((1, 63, 64, 700, 1500))
    dense = _decode(_decoder(model), prompts, 5)
    sparse = _decode(_decoder(model, sparse_attention=SparseAttention(64)), prompts, 5)
    for a, b in zip(sparse, dense):
        _close(a, b)


def _reference_rows(pool, layer, q, cache, setting):
    """Dense attention over the blocks the definition selects, for one single-token row."""
    from tests.test_gpu_sparse_attention import select

    length, heads = cache.length + 1, pool.config.n_kv_heads
    table = torch.tensor([page.index for page in cache.pages], dtype=torch.int32)
    keys, values = pool.keys[layer].cpu(), pool.values[layer].cpu()
    group = q.shape[0] // heads
    out = []
    for h in range(heads):
        query = q[h * group:(h + 1) * group].double()
        count = -(-length // 64)
        bounds = torch.zeros(keys.shape[0], 4, 2, 128)
        for b in range(count):
            part = keys[int(table[b // 4]), 64 * (b % 4):64 * (b % 4) + min(64, length - 64 * b), h]
            bounds[int(table[b // 4]), b % 4, 0], bounds[int(table[b // 4]), b % 4, 1] = part.amin(0), part.amax(0)
        blocks = select(query, bounds, table, length, setting.top_blocks, setting.sink_blocks, setting.recent_blocks)
        at = torch.cat([torch.arange(64 * b, min(length, 64 * b + 64)) for b in blocks])
        k, v = keys[table.long()[at // 256], at % 256, h].double(), values[table.long()[at // 256], at % 256, h].double()
        out.append(torch.softmax(query @ k.t() * 128 ** -0.5, -1) @ v)
    return torch.cat(out)


def test_sparse_rows_of_any_tick():
    """Single-token rows attend to the blocks that the keys in the pool select, in decode ticks and
    beside prefill chunks, after truncation, and over restored pages; other rows stay dense."""
    from helios_b200.paged_cache import PackedBatchCache

    config = Qwen3Config(**{**SHAPE, "n_layers": 1})
    pool = KVPagePool(config, 40, device=DEV)
    setting = SparseAttention(top_blocks=6)
    g = torch.Generator().manual_seed(3)

    def tick(caches, counts, sparse=setting):
        batch = PackedBatchCache(caches)
        batch.sparse = sparse
        batch.prepare_packed(counts)
        total = sum(counts)
        q, k, v = (torch.randn(1, n, total, 128, generator=g).to(torch.bfloat16).to(DEV) for n in (8, 2, 2))
        out = batch.attend(0, q, k, v)
        rows, at = [], 0
        for cache, count in zip(caches, counts):
            if count == 1:
                rows.append((out[0, :, at].cpu().double(), _reference_rows(pool, 0, q[0, :, at].cpu(), cache, setting)))
            at += count
        batch.advance_packed()
        return rows, out, q

    a, b, c = (PagedKVCache(pool, 2000) for _ in range(3))
    tick([a, b], [1100, 700], None)  # before the pool keeps bounds
    pool.enable_key_bounds()
    for counts, caches in (([1, 1], [a, b]), ([1, 300, 1], [a, c, b]), ([1, 1, 1], [a, b, c])):
        rows, _, _ = tick(caches, counts)
        for got, want in rows:
            assert (got - want).abs().max() < 0.02 and want.abs().max() > 0.05
    # Truncated and written again: the old keys' bounds are gone.
    b.truncate(640)
    rows, _, _ = tick([b], [1])
    assert (rows[0][0] - rows[0][1]).abs().max() < 0.02
    # Pages restored by aliasing keep their bounds.
    d = PagedKVCache(pool, 2000)
    d.restore_blocks([a.snapshot_block(0, 1024)])
    rows, _, _ = tick([d, a], [1, 1])
    for got, want in rows:
        assert (got - want).abs().max() < 0.02
    # Copied pages bring them along.
    pool.copy_pages([a.pages[0].index], [pool._free[0]])
    assert torch.equal(pool.bounds[:, pool._free[0]], pool.bounds[:, a.pages[0].index])
    assert _native.device_status() == 0


def test_sparse_needs_bounds():
    from helios_b200.paged_cache import PagedBatchCache

    pool = KVPagePool(Qwen3Config(**{**SHAPE, "n_layers": 1}), 4, device=DEV)
    batch = PagedBatchCache([PagedKVCache(pool, 100)])
    batch.sparse = SparseAttention()
    batch.prepare(1)
    x = torch.zeros(1, 8, 1, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="enable_key_bounds"):
        batch.attend(0, x, x[:, :2], x[:, :2])


@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_controls_steer_sampling(temperature):
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(4, 1000, generator=g).to(torch.bfloat16).to(DEV)
    history = TokenHistory(4, 32, DEV)
    best = logits[0].argmax().item()
    slot = history.open([1, 2, 3])
    history.append([slot], torch.tensor([best], device=DEV))
    allowed = torch.zeros(1000, dtype=torch.bool)
    allowed[[17, 900]] = True
    controls = [LogitControls(presence_penalty=100.0, slot=slot), LogitControls(logit_bias={5: 200.0}),
                LogitControls(allowed=allowed), None]
    samplings = [Sampling(1, temperature, 0.9)] * 4
    before = logits.clone()
    uniforms = torch.full((4,), 0.3)
    ids = sample_rows(logits, samplings, uniforms=uniforms, controls=controls, history=history).tolist()
    assert torch.equal(logits, before)
    assert ids[0] != best and ids[1] == 5 and ids[2] in (17, 900)
    assert ids[3] == sample_rows(logits, samplings, uniforms=uniforms)[3].item()
    assert torch.equal(control_rows(logits, controls, history)[3], logits[3])


def test_rows_without_a_token_give_minus_one():
    x = torch.randn(5, 700, device=DEV).to(torch.bfloat16)
    x[1] = x[2] = x[3] = float("-inf")
    x[4] = float("nan")
    samplings = [GREEDY, GREEDY, Sampling(1, 0.8, 0.9), Sampling(1, 0.8, 1.0), GREEDY]
    ids = sample_rows(x, samplings, uniforms=torch.full((5,), 0.5)).tolist()
    assert ids == [x[0].argmax().item(), -1, -1, -1, -1]


def test_all_together_with_and_without_graphs():
    model = _model(3)
    model.quantize_weights(128)
    prompts = _prompts((1000, 7, 400), seed=9)
    setting = SparseAttention(top_blocks=5)
    runs = []
    for graphs in (False, True):
        model._graphs = None
        if graphs:
            model.enable_cuda_graphs()
        decoder = _decoder(model, sparse_attention=setting)
        history = TokenHistory(4, 2048, DEV)
        slots = [history.open(p) for p in prompts]
        controls = [LogitControls(frequency_penalty=2.0, slot=slots[0]),
                    LogitControls(repetition_penalty=1.3, logit_bias={3: -100.0}, slot=slots[1]), None]
        caches = [PagedKVCache(decoder.page_pool, len(p) + 20) for p in prompts]
        logits = decoder.packed_caches(caches, prompts)
        out, seen = [], []
        for _ in range(12):
            ids = sample_rows(logits, [GREEDY] * 3, controls=controls, history=history)
            history.append(slots, ids)
            out.append(ids.tolist())
            seen.append(logits.clone())
            logits = decoder.decode_caches(caches, ids)
        runs.append((out, seen))
        assert history.tokens[slots[0], 1000:1012].tolist() == [step[0] for step in out]
    for a, b in zip(*(seen for _, seen in runs)):
        _close(b, a)
    assert runs[0][0] == runs[1][0]
    assert _native.device_status() == 0


def test_work_queues_behind_its_stream():
    x = torch.randn(2, 256).to(torch.bfloat16).to(DEV)
    from helios_b200.w4 import quantize_w4

    w = quantize_w4(torch.randn(64, 256, device=DEV))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # 10 ms: what follows on this stream must wait for it
        y = x * 2
        got = ops.linear_w4(y, *w)
    side.synchronize()
    assert torch.equal(got, ops.linear_w4(x * 2, *w))
