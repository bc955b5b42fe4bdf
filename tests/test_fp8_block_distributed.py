"""Block-scaled 8-bit layers on sharded parameters (resident and streamed), under tensor parallelism and with experts spread over ranks."""

import json
from pathlib import Path

import pytest
import torch
import torch.distributed as dist

from olmo_core_b200.float8 import BlockFloat8LinearConfig, Float8Config, refresh_float8_scales
from olmo_core_b200.nn.transformer import TransformerConfig
from olmo_core_b200.optim import AdamWConfig
from olmo_core_b200.testing import run_distributed_test

VOCAB, SEQ = 256, 32


def _float8(hp=False):
    return Float8Config(block=BlockFloat8LinearConfig(wgrad_high_precision=hp), cache_weight_casts=True)


def _model():
    torch.manual_seed(0)
    model = TransformerConfig.olmo2_30M(vocab_size=VOCAB, n_layers=3).build(init_device="cpu")
    torch.manual_seed(0)
    model.init_weights(max_seq_len=SEQ, device=torch.device("cpu"))
    model.apply_fp8(_float8())
    return model


def _batch(seed):
    return torch.randint(0, VOCAB, (2, SEQ), generator=torch.Generator().manual_seed(seed))


def _sharded_worker(param_dtype):
    from olmo_core_b200.parallel.fsdp import ShardedParamRuntime

    rank = dist.get_rank()
    dtype = None if param_dtype is None else getattr(torch, param_dtype)

    def build(**mode):
        model = _model()
        rt = model._sharding_runtime = ShardedParamRuntime(model, param_dtype=dtype, reduce_dtype=torch.float32, **mode)
        rt.materialize(torch.device("cpu"))
        rt.sync_lowp()
        return model, rt

    def step(model, rt):
        rt.zero_grad()
        loss = model(_batch(rank), labels=_batch(rank)).loss
        loss.backward()
        rt.reduce_gradients()
        return float(loss)

    if dtype is None:  # what the two ranks' batches give on a plain model
        plain = _model()
        losses = [plain(_batch(r), labels=_batch(r)).loss for r in range(2)]
        (sum(losses) / 2).backward()
        want_loss, want = float(losses[rank]), {n: p.grad for n, p in plain.named_parameters()}
    else:  # the same arithmetic on whole copies
        model, rt = build(shard=False)
        want_loss, want = step(model, rt), {slot.name: rt.grad_view(slot).clone() for slot in rt.slots}
    for streamed in (False, True):
        model, rt = build(shard=True, streamed=streamed)
        assert rt.streamed == streamed
        optim = AdamWConfig(lr=1e-2).build(model)
        # the same products on the same values: only the order in which two fp32 gradients are averaged differs
        first = step(model, rt)
        assert first == pytest.approx(want_loss, rel=1e-5)
        for slot in rt.slots:
            got, full = rt.grad_view(slot), want[slot.name]
            rows = slice(slot.row_start, slot.row_start + got.shape[0]) if slot.sharded else slice(None)
            err = (got[: full[rows].shape[0]] - full[rows]).norm() / full.norm()
            assert err <= 1e-4, (slot.name, float(err), streamed)
        for _ in range(2):
            optim.step()
            model.post_optim_step()
            loss = step(model, rt)
        assert loss != first  # the updated weights are what runs
        refresh_float8_scales(model)
        assert step(model, rt) == loss  # and nothing older
    dist.barrier()


@pytest.mark.parametrize("param_dtype", [None, "bfloat16"])
def test_sharded_parameters(param_dtype):
    run_distributed_test(_sharded_worker, world_size=2, func_args=(param_dtype,))


def _tensor_parallel_losses(tp, block=True):
    from olmo_core_b200.train.train_module import (
        TransformerDataParallelConfig,
        TransformerTensorParallelConfig,
        TransformerTrainModule,
    )

    torch.manual_seed(0)
    model = TransformerConfig.olmo2_30M(vocab_size=VOCAB, n_layers=2).build(init_device="cpu")
    torch.manual_seed(0)
    model.init_weights(max_seq_len=SEQ, device=torch.device("cpu"))
    model.init_weights = lambda *a, **k: None  # both layouts start from these weights
    module = TransformerTrainModule(
        model=model, optim=AdamWConfig(lr=1e-3, weight_decay=0.0), rank_microbatch_size=4 * SEQ, max_sequence_length=SEQ,
        max_grad_norm=1.0, device=torch.device("cpu"), tp_config=TransformerTensorParallelConfig(degree=2) if tp else None,
        dp_config=TransformerDataParallelConfig(name="ddp") if tp else None, float8_config=_float8() if block else None)
    assert not block or any(getattr(m, "float8", None) is not None for m in module.model.modules())
    gen, out = torch.Generator().manual_seed(7), []
    for _ in range(3):
        ids = torch.randint(0, VOCAB, (4, SEQ), generator=gen)
        module.zero_grads()
        module.train_batch({"input_ids": ids})
        module.optim_step()
        out.append(float(module.latest_ce_loss))
    return out


def _tensor_parallel_worker(path):
    losses = _tensor_parallel_losses(True)
    if dist.get_rank() == 0:
        Path(path).write_text(json.dumps(losses))


def test_tensor_parallel(tmp_path):
    want = _tensor_parallel_losses(False)
    assert want != _tensor_parallel_losses(False, block=False)  # the quantised layers are really in use
    run_distributed_test(_tensor_parallel_worker, world_size=2, func_args=(str(tmp_path / "losses.json"),))
    # partial sums are rounded to bf16 on either rank (2^-8 each) before they are added
    assert json.loads((tmp_path / "losses.json").read_text()) == pytest.approx(want, rel=5e-3)


def _expert_parallel_worker():
    from torch.distributed.device_mesh import init_device_mesh

    from olmo_core_b200.nn.moe.mlp import DroplessMoEMLP
    from olmo_core_b200.nn.moe.parallel_mlp import ParallelDroplessMLP

    rank, ws, E, D, HID, K, N = dist.get_rank(), dist.get_world_size(), 8, 72, 136, 2, 21

    def build():
        torch.manual_seed(0)  # the same full set of experts everywhere
        return ParallelDroplessMLP(mlp=DroplessMoEMLP(d_model=D, hidden_size=HID, num_experts=E, dtype=torch.float32,
                                                      init_device="cpu"), top_k=K)

    full, sharded = build(), build()
    sharded.apply_ep(init_device_mesh("cpu", (ws,), mesh_dim_names=("ep",)))
    for mod in (full, sharded):
        _float8().apply_float8_linear(mod)
        assert mod.mlp.float8 is not None
    gen = torch.Generator().manual_seed(10 + rank)
    for _ in range(2):
        x = torch.randn(1, N, D, generator=gen)
        weights, idx = torch.softmax(torch.randn(N, E, generator=gen), -1).topk(K, dim=-1)
        counts = torch.bincount(idx.reshape(-1), minlength=E)
        results = []
        for mod in (full, sharded):
            xi, wi = x.clone().requires_grad_(True), weights.view(1, N, K).clone().requires_grad_(True)
            y = mod(xi, wi, idx.view(1, N, K), counts)
            y.square().sum().backward()
            results.append((y.detach(), xi.grad, wi.grad))
        for a, b in zip(*results):  # a row's products do not know which other rows there are
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    for name in ("w1", "w2", "w3"):
        g = getattr(full.mlp, name).grad.clone()
        dist.all_reduce(g)  # this rank's experts saw the tokens of both ranks
        rows = g.shape[0] // ws
        torch.testing.assert_close(getattr(sharded.mlp, name).grad, g[rank * rows:(rank + 1) * rows], rtol=1e-4, atol=1e-5)


def test_expert_parallel():
    run_distributed_test(_expert_parallel_worker, world_size=2, backend="gloo")
