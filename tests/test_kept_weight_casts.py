"""8-bit copies of weights that layers keep between calls: they go when the weights change, whichever way that happens."""

from types import SimpleNamespace

import pytest
import torch

from olmo_core_b200.float8 import AOMXLinearConfig, BlockFloat8LinearConfig, Float8Config
from olmo_core_b200.nn.feed_forward import Linear
from olmo_core_b200.nn.transformer import TransformerConfig
from olmo_core_b200.ops import fp8_block as fb

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(seed, device="cpu", dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return TransformerConfig.olmo2_30M(vocab_size=512, n_layers=2).build(init_device="cpu").to(device, dtype)


def _kept(*layers):
    Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True).apply_float8_linear(torch.nn.Sequential(*layers))


def _generation_module(seed, device):
    from olmo_core_b200.generate.generation_module.config import GenerationConfig
    from olmo_core_b200.generate.generation_module.transformer import TransformerGenerationModule

    return TransformerGenerationModule(
        _model(seed), GenerationConfig(max_new_tokens=4, do_sample=False, use_cache=True, pad_token_id=0, eos_token_id=511),
        float8_config=Float8Config(block=BlockFloat8LinearConfig()), device=torch.device(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("in_place", [False, True])
def test_generation_after_other_weights_were_loaded(in_place, device):
    module, fresh = _generation_module(0, device), _generation_module(1, device)
    ids = torch.randint(1, 500, (2, 9), device=device)
    before, logits_before, _ = module.generate_batch(ids, return_logits=True, log_timing=False)
    state = fresh.state_dict()
    if in_place:  # as a checkpoint reader does: the module's own memory is written, then handed back
        own = module.state_dict()
        for name, value in state["model"].items():
            own["model"][name].copy_(value)
        state = own
    module.load_state_dict(state)
    got, logits, _ = module.generate_batch(ids, return_logits=True, log_timing=False)
    want, want_logits, _ = fresh.generate_batch(ids, return_logits=True, log_timing=False)
    assert torch.equal(got, want) and torch.equal(logits, want_logits)
    assert not torch.equal(logits, logits_before)


def _train_module(seed):
    from olmo_core_b200.optim import AdamWConfig
    from olmo_core_b200.train.train_module import TransformerTrainModuleConfig

    module = TransformerTrainModuleConfig(
        rank_microbatch_size=64, max_sequence_length=32, optim=AdamWConfig(lr=1e-3),
        float8_config=Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True)).build(
            _model(seed, dtype=torch.float32), device=torch.device("cpu"))
    with torch.no_grad():
        for p in module.model.parameters():
            p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(seed)) * 0.05)
    return module


def test_training_module_after_a_checkpoint_was_loaded():
    module, other = _train_module(0), _train_module(1)
    ids = torch.randint(1, 500, (2, 9))
    with torch.no_grad():
        before = module.model(ids)
        module.load_state_dict({"model": other.state_dict(optim=False)["model"]})
        got, want = module.model(ids), other.model(ids)
    assert torch.equal(got, want) and not torch.equal(got, before)


def test_merged_weights_are_evaluated_and_leave_nothing_behind(tmp_path, monkeypatch):
    from olmo_core_b200.train.callbacks import model_merger
    from olmo_core_b200.train.callbacks.model_merger import ModelMergeCallback

    module, other = _train_module(0), _train_module(1)
    ids = torch.randint(1, 500, (2, 9))
    seen = []

    def evaluate(self):
        with torch.no_grad():
            seen.append(module.model(ids))

    monkeypatch.setattr(model_merger, "save_state_dict", lambda *args, **kwargs: None)
    monkeypatch.setattr(ModelMergeCallback, "_evaluate_merged", evaluate)
    callback = ModelMergeCallback(merge_step=1, merge_last_n_steps=1)
    callback.trainer = SimpleNamespace(train_module=module, checkpointer=SimpleNamespace(process_group=None), save_folder=str(tmp_path))
    monkeypatch.setattr(ModelMergeCallback, "_merged_checkpoint_path", lambda self, step: str(tmp_path / "merged"))
    callback._accumulators = {1: {n: p.detach().clone() for n, p in other.model.named_parameters()}}
    callback._accumulator_counts = {1: 1}
    with torch.no_grad():
        live = module.model(ids)
        merged = other.model(ids)
        callback._save_merged_checkpoint(1)
        again = module.model(ids)
    assert torch.equal(seen[0], merged) and torch.equal(again, live) and not torch.equal(live, merged)


@pytest.mark.parametrize("device", DEVICES)
def test_a_replaced_or_moved_weight_is_cast_again(device):
    lin = Linear(64, 64, False, torch.bfloat16, "cpu").to(device)
    _kept(lin)
    x = torch.randn(7, 64, device=device, dtype=torch.bfloat16)
    lin(x)
    for change in (lambda w: torch.randn_like(w), lambda w: w.t(), lambda w: w.float() * 3):
        lin.weight.data = change(lin.weight.data)
        assert torch.equal(lin(x), fb.fp8_block_linear(x, lin.weight))
    version, kept = lin.weight._version, lin.float8["weight_cache"]["block_tiles"]
    lin(x)
    assert lin.weight._version == version and lin.float8["weight_cache"]["block_tiles"] is kept  # nothing changed: nothing made


@pytest.mark.gpu
def test_a_layer_moved_to_the_host_and_back():
    lin = Linear(64, 48, False, torch.bfloat16, "cpu").to("cuda")
    _kept(lin)
    x = torch.randn(7, 64, device="cuda", dtype=torch.bfloat16)
    want = lin(x)
    lin.to("cpu")
    assert torch.equal(lin(x.cpu()), fb.fp8_block_linear(x.cpu(), lin.weight))
    lin.to("cuda")
    assert torch.equal(lin(x), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("config", [Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True),
                                    Float8Config(ao_mx=AOMXLinearConfig.mxfp8_cublas_rceil(), cache_weight_casts=True)])
def test_weights_made_under_inference_mode_are_not_kept(config, device):
    with torch.inference_mode():
        lin = Linear(256, 128, False, torch.bfloat16, "cpu").to(device)
        config.apply_float8_linear(torch.nn.Sequential(lin))
        x = torch.randn(128, 256, device=device, dtype=torch.bfloat16)
        first = lin(x)
        lin.weight.mul_(2)  # counts no version
        assert torch.equal(lin(x), 2 * first)


def _captured(fn):
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = fn()
    return graph, out


@pytest.mark.gpu
@pytest.mark.parametrize("config", [Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True),
                                    Float8Config(ao_mx=AOMXLinearConfig.mxfp8_cublas_rceil(), cache_weight_casts=True)])
def test_what_a_graph_makes_is_not_kept(config):
    lin = Linear(256, 128, False, torch.bfloat16, "cpu").to("cuda")
    config.apply_float8_linear(torch.nn.Sequential(lin))
    x = torch.randn(128, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want = lin(x).clone()
        lin.float8["weight_cache"].clear()
        graph, out = _captured(lambda: lin(x))
        assert not lin.float8["weight_cache"]
        assert torch.equal(lin(x), want)  # before the first replay
        graph.replay()
        assert torch.equal(out, want)
        del graph, out  # what eager calls kept does not depend on it
        torch.empty(1 << 26, device="cuda").fill_(float("nan"))
        assert torch.equal(lin(x), want)


@pytest.mark.gpu
def test_a_kept_cast_outlives_its_place_in_the_cache_for_a_graph_that_reads_it():
    from olmo_core_b200.float8 import refresh_float8_scales

    lin = Linear(256, 128, False, torch.bfloat16, "cpu").to("cuda")
    _kept(lin)
    x = torch.randn(3, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want = lin(x).clone()
        graph, out = _captured(lambda: lin(x))
        lin.weight.mul_(2)
        refresh_float8_scales(lin)
        assert torch.equal(lin(x), 2 * want)
        torch.cuda.synchronize()
        junk = [torch.full_like(lin.float8["weight_cache"]["block_tiles"][1], 0x7F) for _ in range(64)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and len(junk) == 64


@pytest.mark.gpu
@pytest.mark.parametrize("config", [Float8Config(block=BlockFloat8LinearConfig(), cache_weight_casts=True),
                                    Float8Config(ao_mx=AOMXLinearConfig.mxfp8_cublas_rceil(), cache_weight_casts=True)])
def test_another_stream_waits_for_the_cast_that_it_uses(config):
    lin = Linear(1024, 512, False, torch.bfloat16, "cpu").to("cuda")
    x = torch.randn(128, 1024, device="cuda", dtype=torch.bfloat16)
    config.apply_float8_linear(torch.nn.Sequential(lin))
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = lin(x).clone()
        with torch.cuda.stream(two):
            lin(x)  # its own buffers are warm
        lin.float8["weight_cache"].clear()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            junk = [torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") for n in (512 * 1024 + 4 * 32, 512 * 1024, 512 * 32)]
            del junk  # what this stream allocates next holds no weights
            torch.cuda._sleep(20_000_000)  # about 10 ms
            first = lin(x)
        with torch.cuda.stream(two):
            second = lin(x)
        torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("device", DEVICES)
def test_layers_with_kept_casts_can_be_copied_and_pickled(device):
    import copy
    import pickle

    lin = Linear(64, 48, False, torch.bfloat16, "cpu").to(device)
    _kept(lin)
    x = torch.randn(7, 64, device=device, dtype=torch.bfloat16)
    want = lin(x)
    for other in (copy.deepcopy(lin), pickle.loads(pickle.dumps(lin))):
        assert torch.equal(other(x), want)
        with torch.no_grad():
            other.weight.mul_(2)
        assert torch.equal(other(x), 2 * want) and torch.equal(lin(x), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["AdamWConfig", "SkipStepAdamWConfig", "AdamConfig", "LionConfig", "SkipStepLionConfig", "MuonConfig"])
def test_an_optimizer_step_alone_drops_the_casts(name, device):
    import olmo_core_b200.optim as optim

    lin = Linear(64, 48, False, torch.float32, "cpu").to(device)
    _kept(lin)
    optimizer = getattr(optim, name)(lr=0.1).build(lin)
    x = torch.randn(7, 64, device=device, dtype=torch.bfloat16)
    for _ in range(2):
        if hasattr(optimizer, "latest_loss"):
            optimizer.latest_loss = torch.tensor(1.0, device=device)
        y = lin(x)
        y.float().square().sum().backward()
        optimizer.step()
        optimizer.zero_grad()
        after = lin(x)
        assert torch.equal(after, fb.fp8_block_linear(x, lin.weight)) and not torch.equal(after, y)
