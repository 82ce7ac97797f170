"""Sliding window + sinks and the 4-bit KV cache as they are used: training, generation, the command lines."""
import json
import math

import pytest
import torch

from finetune_controller_amd import ops
from finetune_controller_amd.models import LoRAConfig, build_model
from finetune_controller_amd.models.config import ModelConfig, get_config
from finetune_controller_amd.models.generate import generate
from finetune_controller_amd.ops import kv4
from finetune_controller_amd.ops.decode import decode_attention_reference, visible_keys
from finetune_controller_amd.train.trainer import TrainConfig, Trainer

from test_distributed import _hold, _rank_env, _run_ranks

CFG = dict(family="llama", vocab_size=384, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512, max_seq_len=512)


def _model(dev="cpu", dtype=torch.float32, lora=None, **kw):
    torch.manual_seed(0)
    m = build_model(ModelConfig(**{**CFG, **kw}), lora, device=dev, dtype=dtype)
    m.init_weights(seed=4, std=0.06)
    return m.eval()


def _prompts(vocab, lens=(5, 17, 60)):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(3, vocab, (n,), generator=g).tolist() for n in lens]


# ---------------------------------------------------------------- configuration
def test_config_options(tmp_path):
    c = get_config("mistral-tiny", attention_sinks=4)
    assert (c.sliding_window, c.attention_sinks) == (64, 4)
    assert get_config("llama-tiny", 32, 2).sliding_window == 32 and get_config("mistral-tiny", 0).sliding_window == 0
    (tmp_path / "c.json").write_text(json.dumps(c.to_hf_config()))
    r = get_config(str(tmp_path / "c.json"))
    assert (r.sliding_window, r.attention_sinks) == (64, 4)
    assert "attention_sinks" not in get_config("mistral-tiny").to_hf_config()
    for bad in (("llama-tiny", -1, 2), ("gpt2-tiny", 8, 0), ("mistral-tiny", 0, 1)):
        with pytest.raises(ValueError):
            get_config(*bad)


def test_job_spec_passes_the_options():
    from finetune_controller_amd.controlplane.spec.models.builtin import Llama3_8B_LoRA

    spec = Llama3_8B_LoRA()
    spec.training_arguments.sliding_window, spec.training_arguments.attention_sinks = 1024, 4
    cmd = spec.run_cmd()[-1]
    assert "--sliding-window=1024" in cmd and "--attention-sinks=4" in cmd
    from finetune_controller_amd.train.cli import build_parser, config_from_args

    tc = config_from_args(build_parser().parse_args(["--sliding-window=1024", "--attention-sinks=4"]))
    assert (tc.sliding_window, tc.attention_sinks) == (1024, 4)


# ---------------------------------------------------------------- bf16 / fp32 cache with sinks
def test_decode_reference_with_sinks():
    B, L, H, KV, D = 4, 40, 4, 2, 16
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(B, H * D, generator=g), torch.randn(B, L, KV * D, generator=g), torch.randn(B, L, KV * D, generator=g)
    lens = torch.tensor([40, 7, 23, 1], dtype=torch.int32)
    out = decode_attention_reference(q, k, v, lens, H, KV, D, 0.25, window=10, sinks=3)
    for b in range(B):
        n = int(lens[b])
        idx = [t for t in range(n) if t >= n - 10 or t < 3]
        assert visible_keys(lens, L, 10, 3)[b].nonzero().flatten().tolist() == idx
        for h in range(H):
            c = slice(h // 2 * D, (h // 2 + 1) * D)
            p = (k[b, idx, c] @ q[b, h * D:(h + 1) * D] * 0.25).softmax(0)
            torch.testing.assert_close(out[b, h * D:(h + 1) * D], p @ v[b, idx, c], atol=1e-5, rtol=1e-5)
    with pytest.raises(ValueError, match="sinks"):
        ops.decode_attention(torch.zeros(B, 8 * D), k, v, lens, L, H, KV, D, sinks=-1)


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KV,window,sinks", [(128, 8, 2, 100, 4), (64, 8, 8, 1, 70), (128, 4, 1, 300, 300), (64, 4, 2, 0, 9)])
def test_decode_kernel_with_sinks(D, H, KV, window, sinks):
    B, L = 3, 700
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(B, (H + 2 * KV) * D, generator=g).bfloat16()
    k, v = (torch.randn(B, L, KV * D, generator=g).bfloat16() for _ in range(2))
    lens = torch.tensor([700, 1, 333], dtype=torch.int32)
    got = ops.decode_attention(qkv.cuda(), k.cuda(), v.cuda(), lens.cuda(), L, H, KV, D, window=window, sinks=sinks)
    for b in range(B):
        k[b, lens[b] - 1], v[b, lens[b] - 1] = qkv[b, H * D:(H + KV) * D], qkv[b, (H + KV) * D:]
    args = (lens, H, KV, D, D ** -0.5, window, sinks)
    want = decode_attention_reference(qkv.double(), k, v, *args).double()
    pv = decode_attention_reference(qkv.double(), k, v.abs(), *args).double()
    # the output's rounding; scores, weights and sums in 32 bits (the oracle's too)
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * pv).all()


# ---------------------------------------------------------------- generation
@pytest.mark.parametrize("sinks", [1, 5])
def test_cached_greedy_with_sinks_matches_recompute(sinks):
    m = _model(sliding_window=24, attention_sinks=sinks)
    for p, o in zip(_prompts(384), generate(m, _prompts(384), max_new_tokens=20)):
        ids = list(p)
        for t in o:
            with torch.no_grad():
                assert t == int(m(torch.tensor([ids]))[-1].argmax())
            ids.append(t)


class _Held(ops.KVCache):
    """A plain cache whose rows went through the 4-bit format: what KV4Cache has to equal."""

    def _hold(self, t):
        c, s = kv4.quantize_reference(t.unflatten(-1, (self.KV, self.D)))
        return kv4._held(c, s).flatten(-2)

    def store(self, layer, qkv, H, S):
        q = qkv.clone()
        q[:, H * self.D:] = torch.cat([self._hold(x) for x in q[:, H * self.D:].chunk(2, 1)], 1)
        super().store(layer, q, H, S)

    def attend(self, layer, qkv, H, window=0, sinks=0):
        q = qkv.clone()
        q[:, H * self.D:] = torch.cat([self._hold(x) for x in q[:, H * self.D:].chunk(2, 1)], 1)
        return super().attend(layer, q, H, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_generate_with_a_4_bit_cache(monkeypatch, window, sinks):
    m = _model(sliding_window=window, attention_sinks=sinks)
    got = generate(m, _prompts(384), max_new_tokens=16, kv_bits=4)
    monkeypatch.setattr(ops, "KVCache", _Held)
    assert got == generate(m, _prompts(384), max_new_tokens=16)
    with pytest.raises(ValueError, match="kv_bits"):
        generate(m, _prompts(384), kv_bits=8)
    tiny = build_model(get_config("llama-tiny"), None, device="cpu", dtype=torch.float32)  # head_dim 32
    tiny.init_weights(seed=1)
    with pytest.raises(ValueError, match="head_dim"):
        generate(tiny, [[5, 6]], kv_bits=4)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,window,sinks", [((4, 2), 0, 0), ((2, 1), 100, 4)])
def test_gpu_generation_steps(heads, window, sinks, monkeypatch):
    """Cached decode steps on the GPU kernels (D = 64 / 128): logits against re-running the sequence; the 4-bit cache
    against the plain cache of the same quantised rows; captured steps equal eager ones."""
    monkeypatch.setenv("FTC_KERNELS", "hip")
    m = _model("cuda", torch.bfloat16, n_heads=heads[0], n_kv_heads=heads[1], sliding_window=window, attention_sinks=sinks,
               dim=256)
    cfg = m.cfg
    ids = torch.randint(3, 384, (1, 300), generator=torch.Generator().manual_seed(1)).cuda()
    n = len(m.layers)
    caches = [ops.KVCache(n, 1, 320, cfg.n_kv_heads, cfg.head_dim, "cuda"), _Held(n, 1, 320, cfg.n_kv_heads, cfg.head_dim, "cuda"),
              ops.KV4Cache(n, 1, 320, cfg.n_kv_heads, cfg.head_dim, "cuda")]
    logits = []
    with torch.no_grad():
        for c in caches:
            c.row = 0
            m.hidden(ids[:, :296], kv_cache=c)
            c.finish_prefill(0, 296)
            out = []
            for t in range(296, 300):
                pos = c.begin_decode()
                x = m.hidden(ids[:, t:t + 1], positions=pos, kv_cache=c)
                c.end_decode()
                c.decoding = False
                out.append((x @ m.lm_head.t()).float()[-1])
            logits.append(torch.stack(out))
        full = torch.stack([m(ids[:, :t + 1]).float()[-1] for t in range(296, 300)])
    plain, held, four = logits
    # bf16 activations re-associated by other kernels: a few roundings (2^-8) of the largest logit
    assert (plain - full).abs().max() <= 0.03 * full.abs().max() + 0.03
    assert (four - held).abs().max() <= 0.03 * held.abs().max() + 0.03
    assert (four - plain).norm() <= 0.2 * plain.norm()  # what 4 bits cost here
    prompts = _prompts(384, (9, 40, 130))
    for bits in (16, 4):
        eager = generate(m, prompts, max_new_tokens=12, kv_bits=bits, graph=False)
        assert generate(m, prompts, max_new_tokens=12, kv_bits=bits, graph=True) == eager


# ---------------------------------------------------------------- training
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("method", ["lora", "full"])
def test_train_with_sinks_then_generate_from_the_artifacts(tmp_path, capsys, dev, method):
    """The worker's path: fine-tune with a window and sinks, save, continue a prompt with the 4-bit cache."""
    cfg = ModelConfig(**{**CFG, "n_heads": 2, "n_kv_heads": 1}, sliding_window=16, name="t")
    (tmp_path / "m.json").write_text(json.dumps(cfg.to_hf_config()))
    out = tmp_path / "out"
    tr = Trainer(TrainConfig(model=str(tmp_path / "m.json"), method=method, batch_size=2, seq_len=75, synthetic=True, max_steps=2,
                             checkpoint_path=str(out), resume=False, device=dev, lr=1e-3, warmup_steps=0, attention_sinks=3))
    assert tr.cfg.attention_sinks == 3
    tr.run()
    tr.close()
    from finetune_controller_amd.models.generate import main

    capsys.readouterr()
    src = ["--adapter", str(out), "--model", str(tmp_path / "m.json")] if method == "lora" else \
        ["--init-from", str(out), "--model", str(out / "config.json")]
    if method == "full":
        assert get_config(str(out / "config.json")).attention_sinks == 3
    assert main([*src, "--prompt", "hi", "--max-new-tokens", "4", "--kv-bits", "4", "--attention-sinks", "3"]) == 0
    assert capsys.readouterr().out.startswith("hi")


def test_packed_documents_with_sinks_are_refused(tmp_path):
    with pytest.raises(ValueError, match="pack_documents"):
        Trainer(TrainConfig(model="mistral-tiny", attention_sinks=2, pack_documents=True, synthetic=True, device="cpu",
                            checkpoint_path=str(tmp_path)))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [256, 300])
def test_model_gradients_match_the_torch_path(S, monkeypatch):
    """LoRA gradients of a whole decoder with sinks (RoPE handed to the attention backward, padded buffers of the
    augmented projections) against the torch path in 32 bits."""
    ref = _model(lora=LoRAConfig(r=16, alpha=32), n_heads=2, n_kv_heads=1, sliding_window=60, attention_sinks=4)
    for layer in ref.layers:
        for i, pair in enumerate(layer.lora.values()):
            for _, _, b in pair.segment_tensors():  # (the blocks off the diagonal stay zero)
                b.data.copy_(torch.randn(b.shape, generator=torch.Generator().manual_seed(i)) * 0.02)
    weights = {k: v.bfloat16().float() for k, v in ref.state_dict().items()}

    def grads(dev, dtype, mode):
        monkeypatch.setenv("FTC_KERNELS", mode)
        m = _model(dev, dtype, lora=LoRAConfig(r=16, alpha=32), n_heads=2, n_kv_heads=1, sliding_window=60, attention_sinks=4)
        m.load_state_dict(weights)
        m.invalidate_transposed()
        m.train()
        m.freeze_base()
        ids = torch.randint(3, 384, (2, S), generator=torch.Generator().manual_seed(5)).to(dev)
        m(ids, ids.roll(-1, 1)).backward()
        return torch.cat([(p.grad if p.grad is not None else p.main_grad).float().cpu().flatten()
                          for _, p in m.named_parameters() if p.requires_grad])

    want = grads("cpu", torch.float32, "torch")
    got = grads("cuda", torch.bfloat16, "hip")
    cos = torch.nn.functional.cosine_similarity(got.double(), want.double(), dim=0)
    assert cos > 0.998 and abs(float(got.norm() / want.norm()) - 1) < 0.03, float(cos)


def _sp_worker(rank, world, port, tmp, q):
    _rank_env(rank, world, port, tmp)
    tr = Trainer(_sp_config(tmp, world))
    loss = tr.train_step(0.0)
    q.put((rank, {"loss": float(loss), "grad": tr.opt.grad_flat.detach().double().clone()}))
    tr.close()
    _hold(tmp, port)


def _sp_config(tmp, sp):
    return TrainConfig(model="mistral-tiny", method="full", batch_size=2, seq_len=64, synthetic=True, max_steps=1,
                       checkpoint_path=str(tmp), resume=False, device="cpu", dtype="fp32", lr=0.0, max_grad_norm=0.0,
                       save_model=False, sp=sp, bucket_mb=0.05, sliding_window=20, attention_sinks=3)


@pytest.mark.slow
def test_sequence_parallel_with_sinks_matches_a_single_process(tmp_path):
    res = _run_ranks(_sp_worker, 2, tmp_path)
    tr = Trainer(_sp_config(tmp_path, 1))
    ref_loss, ref = float(tr.train_step(0.0)), tr.opt.grad_flat.detach().double().clone()
    tr.close()
    assert abs((res[0]["loss"] + res[1]["loss"]) / 2 - ref_loss) < 1e-5 * abs(ref_loss)
    torch.testing.assert_close(res[0]["grad"] / 2, ref, atol=1e-6 * ref.abs().max().item(), rtol=1e-4)
    assert not math.isnan(ref_loss)


@pytest.mark.parametrize("model,trained", [("llama-tiny", (16, 3)), ("mistral-tiny", (0, -1)), ("mistral-tiny", (-1, 2)),
                                           ("llama-tiny", (-1, -1))])
def test_an_adapter_keeps_the_attention_it_was_trained_with(tmp_path, monkeypatch, model, trained):
    """Generation from a LoRA adapter without flags sees what training saw; flags still replace it."""
    from finetune_controller_amd.models import checkpoint as ckpt
    from finetune_controller_amd.models import generate as gen

    tr = Trainer(TrainConfig(model=model, method="lora", batch_size=1, seq_len=32, synthetic=True, max_steps=1, resume=False,
                             checkpoint_path=str(tmp_path / "out"), device="cpu", sliding_window=trained[0],
                             attention_sinks=trained[1]))
    want = (tr.cfg.sliding_window, tr.cfg.attention_sinks)
    tr.run()
    ckpt.save_adapter(tr.model, str(tmp_path / "saved"), model, tr.lora)  # by itself, without the trainer's records
    tr.close()
    used = []

    def seen(m, *a, **k):
        used.append((m.cfg.sliding_window, m.cfg.attention_sinks))
        return [[5]]

    monkeypatch.setattr(gen, "generate", seen)
    (tmp_path / "older").mkdir()  # an adapter that has the trainer's record only
    for f in ("adapter_config.json", "adapter_model.safetensors", "training_config.json"):
        (tmp_path / "older" / f).write_bytes((tmp_path / "out" / f).read_bytes())
    for d in ("out", "saved", "older"):
        assert gen.main(["--model", model, "--adapter", str(tmp_path / d), "--prompt", "a"]) == 0
        assert used.pop() == want, d
    flags = ["--sliding-window", "9", "--attention-sinks", "1"]
    assert gen.main(["--model", model, "--adapter", str(tmp_path / "out"), "--prompt", "a", *flags]) == 0
    assert used.pop() == (9, 1)
    conf = json.load(open(tmp_path / "out" / "adapter_config.json"))
    assert not {"sliding_window", "attention_sinks"} & set(conf)  # the PEFT file holds PEFT's keys only
    (tmp_path / "older" / "training_config.json").unlink()  # neither record: the model's own
    assert gen.main(["--model", model, "--adapter", str(tmp_path / "older"), "--prompt", "a"]) == 0
    own = get_config(model)
    assert used.pop() == (own.sliding_window, own.attention_sinks)


def test_full_causal_attention_of_a_model_with_sinks(tmp_path):
    """A window of 0 takes the model's own sinks with it; sinks that are asked for still need a window."""
    (tmp_path / "c.json").write_text(json.dumps(get_config("mistral-tiny", attention_sinks=4).to_hf_config()))
    c = get_config(str(tmp_path / "c.json"), sliding_window=0)
    assert (c.sliding_window, c.attention_sinks) == (0, 0)
    c = get_config(str(tmp_path / "c.json"), sliding_window=30)
    assert (c.sliding_window, c.attention_sinks) == (30, 4)
    with pytest.raises(ValueError, match="needs a sliding window"):
        get_config(str(tmp_path / "c.json"), sliding_window=0, attention_sinks=4)


@pytest.mark.parametrize("why", ["head_dim", "positions"])
def test_a_refused_generation_leaves_the_model_in_its_mode(why):
    m = build_model(get_config("llama-tiny"), None, device="cpu", dtype=torch.float32).train()  # head_dim 32, 512 positions
    kw = dict(kv_bits=4) if why == "head_dim" else dict(max_new_tokens=600)
    with pytest.raises(ValueError, match=why):
        generate(m, [[5, 6]], **kw)
    assert m.training


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_gpu_generation_on_the_torch_path(bits, window, sinks, monkeypatch):
    """FTC_KERNELS=torch: decode steps are captured by default there too, and a captured step equals an eager one."""
    monkeypatch.setenv("FTC_KERNELS", "torch")
    m = _model("cuda", torch.float32, sliding_window=window, attention_sinks=sinks)
    eager = generate(m, _prompts(384), max_new_tokens=10, kv_bits=bits, graph=False)
    assert generate(m, _prompts(384), max_new_tokens=10, kv_bits=bits) == eager


@pytest.mark.gpu
def test_allocations_are_seen_by_dispatch_modes():
    """A mode that follows allocations (a memory tracker) sees what the operators return."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Allocated(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.at = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor) and "empty" in str(func):
                self.at.add(out.untyped_storage().data_ptr())
            return out

    H, KV, D, n = 2, 1, 64, 40
    bf, i32 = dict(dtype=torch.bfloat16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    x = torch.randn(n, (H + 2 * KV) * D, **bf).requires_grad_()
    data, start = ops.kv4_alloc(1, 64, KV, D, device="cuda"), torch.zeros(1, **i32)
    with Allocated() as seen:
        o = ops.attention_packed(x, 1, n, H, KV, D, window=9, sinks=2)
        (g,) = torch.autograd.grad(o, x, torch.ones_like(o))
        alone = ops.attention_packed(x.detach(), 1, n, H, KV, D, window=9, sinks=2)
        rows = ops.kv4_load(data, start, 5, D)
        new = ops.decode_attention_kv4(x.detach()[:1], data, start + 1, 64, H, KV, D)
    assert [t.untyped_storage().data_ptr() in seen.at for t in (o, g, alone, *rows, new)] == [True] * 6


@pytest.mark.parametrize("record", [{"model": "some/base"}, [1], {"model": {"sliding_window": None}}, {}])
def test_records_of_other_tools_say_nothing_of_the_attention(tmp_path, record):
    from finetune_controller_amd.models.checkpoint import adapter_attention

    (tmp_path / "training_config.json").write_text(json.dumps(record))
    assert adapter_attention(str(tmp_path)) == (-1, -1)
