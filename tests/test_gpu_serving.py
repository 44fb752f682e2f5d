"""GPU tests of the low-bit serving path on small random-init models: the 4-bit cache behind HF's own forward and
generate, the 8-bit projections, and both together after a TileMix prefill."""
import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM, Qwen2Config, Qwen2ForCausalLM

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    from tilemix_b200.attention.tilemix import device_error_code

    if torch.cuda.is_available():
        device_error_code()
    yield
    if torch.cuda.is_available():
        assert device_error_code() == 0


# Two runs of a model that differ by fp16 rounding. The attention's output differs by its rounding in either run and the
# operands' in one (3 half steps, 2^-11 each), and each of the nine operations behind it (output projection, residual, norm,
# gate and up, product, down, residual, norm, head) may round to the other side: 12 * 2^-11.
SAME_CODES = 12 * 2.0 ** -11
# A second layer's keys and values are then made from inputs that are apart by up to e = 4 * 2^-11 (2^-9), and a 4-bit code
# flips where a value lies within e |x| of a border: with steps of 1/15 of the range of 32 normal values, 4.1 / 15 = 0.27
# sigma, and |x| = 0.8 sigma on average, in a share 2 * 0.8 e / 0.27 = 6 e of them, by a whole step: 0.27 sqrt(6 e) = 2.9 %
# of the new tokens' keys and values, and at most that of the logits (attention is a part of the residual).
FLIPPED_CODES = 0.03


def _model(dev, kind="llama", head_dim=64, layers=2):
    kw = dict(hidden_size=256, intermediate_size=320, num_hidden_layers=layers, num_attention_heads=4, num_key_value_heads=2,
              vocab_size=300, max_position_embeddings=4096, head_dim=head_dim)
    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(**kw)) if kind == "llama" else Qwen2ForCausalLM(Qwen2Config(**kw))
    return model.to(dev, torch.float16).eval()


def _inject(model, kind="llama"):
    from tilemix_b200.models import tilemix_llama, tilemix_qwen

    module = tilemix_llama if kind == "llama" else tilemix_qwen
    getattr(module, f"inject_tilemix_into_{kind}")(model)
    return module.configure_tilemix_attention_pattern(model, "zero")


def _ids(dev, b, t, seed):
    return torch.randint(0, 300, (b, t), generator=torch.Generator().manual_seed(seed)).to(dev)


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("layers", [1, 2])
@pytest.mark.parametrize("kind", ["llama", "qwen"])
@pytest.mark.parametrize("prompt", [3, 40, 200])
def test_decode_over_the_cache_equals_attention_over_its_values(cuda_device, kind, prompt, layers):
    """A TileMix model that attends in 4 bits against HF's attention given the same cache's values: prompt, single
    tokens, several tokens, a long continuation. One layer sees the same inputs in both and so holds the same codes."""
    from tilemix_b200.models.kv4_cache import Kv4Cache

    plain, tile = _model(cuda_device, kind, layers=layers), _inject(_model(cuda_device, kind, layers=layers), kind)
    bound = SAME_CODES if layers == 1 else FLIPPED_CODES
    cache, ref_cache = Kv4Cache(400, page_size=16), Kv4Cache(400, page_size=32)
    for i, t in enumerate((prompt, 1, 1, 5, 20, 1)):
        ids = _ids(cuda_device, 3, t, seed=i)
        with torch.no_grad():
            got = tile(ids, past_key_values=cache, use_cache=True).logits
            ref = plain(ids, past_key_values=ref_cache, use_cache=True).logits
        assert cache.get_seq_length() == ref_cache.get_seq_length()
        # the first pass of a long prompt sees unrounded keys and values in one model, the cache's in the other
        assert _rel(got, ref) < (bound if i > 0 or prompt < 16 else 0.2), (i, t, _rel(got, ref))
        if i == 0 and prompt >= 16:  # ... and its hidden states of later layers are cached: go on from equal ones
            for a, b in zip(cache.layers, ref_cache.layers):
                k, v = torch.randn((2, 3 * prompt, 2, 64), generator=torch.Generator().manual_seed(9)).half().to(cuda_device)
                from tilemix_b200.attention.kv4 import kv4_append

                kv4_append(k, v, a.pool, cache._all_slots())
                kv4_append(k, v, b.pool, ref_cache._all_slots())


def test_decode_of_a_padded_batch(cuda_device):
    """Short left-padded prompts: padded keys are left out, a request's logits are those it has alone."""
    from tilemix_b200.models.kv4_cache import Kv4Cache

    model = _inject(_model(cuda_device))
    ids, pad = _ids(cuda_device, 2, 9, seed=1), 4
    mask = torch.ones((2, 9), dtype=torch.long, device=cuda_device)
    mask[1, :pad] = 0
    positions = (mask.cumsum(1) - 1).clamp(min=0)
    both, alone = Kv4Cache(64, page_size=16), Kv4Cache(64, page_size=16)
    with torch.no_grad():
        got = model(ids, attention_mask=mask, position_ids=positions, past_key_values=both, use_cache=True).logits[1, -1]
        ref = model(ids[1:, pad:], past_key_values=alone, use_cache=True).logits[0, -1]
        assert _rel(got, ref) < FLIPPED_CODES
        nxt = _ids(cuda_device, 2, 1, seed=2)
        mask = torch.cat([mask, mask[:, -1:]], 1)
        got = model(nxt, attention_mask=mask, position_ids=mask.sum(1, keepdim=True) - 1, past_key_values=both,
                    use_cache=True).logits[1, -1]
        ref = model(nxt[1:], past_key_values=alone, use_cache=True).logits[0, -1]
    assert _rel(got, ref) < FLIPPED_CODES


def test_generate_and_reset(cuda_device):
    from tilemix_b200.models.kv4_cache import Kv4Cache

    model = _inject(_model(cuda_device))
    cache = Kv4Cache(80, page_size=16)
    ids = _ids(cuda_device, 2, 30, seed=3)
    first = model.generate(ids, past_key_values=cache, max_new_tokens=12, do_sample=False, pad_token_id=0)
    assert first.shape == (2, 42) and cache.get_seq_length() == 41
    cache.reset()
    assert cache.get_seq_length() == 0
    again = model.generate(ids, past_key_values=cache, max_new_tokens=12, do_sample=False, pad_token_id=0)
    assert torch.equal(first, again)


def test_cache_refusals(cuda_device):
    from tilemix_b200.models.kv4_cache import Kv4Cache

    for bad in (dict(max_cache_len=0), dict(max_cache_len=10, page_size=8)):
        with pytest.raises(ValueError):
            Kv4Cache(**bad)
    k = torch.zeros((2, 2, 10, 64), dtype=torch.float16, device=cuda_device)
    cache = Kv4Cache(16, page_size=16)
    with pytest.raises(TypeError, match="float16"):
        cache.update(k.float(), k.float(), 0)
    cache.update(k, k, 0)
    with pytest.raises(ValueError, match="same tokens"):
        cache.update(k[:, :, :3], k[:, :, :3], 1)
    with pytest.raises(ValueError, match="max_cache_len"):
        cache.update(k, k, 0)
    with pytest.raises(ValueError, match="2 requests"):
        cache.update(k[:1, :, :1], k[:1, :, :1], 0)
    with pytest.raises(NotImplementedError):
        cache.crop(3)
    with pytest.raises(NotImplementedError):
        cache.reorder_cache(torch.tensor([1, 0]))
    small = Kv4Cache(64, page_size=16, num_pages=3)
    small.append(k, k, 0)
    with pytest.raises(ValueError, match="4 pages"):
        small.append(k, k, 0)


def _dequantised(model, dtype):
    """The model with each projection's weight replaced by what its 8-bit codes stand for."""
    from tilemix_b200.linear.int8_linear import quantize_per_token_int8

    for layer in model.model.layers:
        for m in list(layer.self_attn.children()) + list(layer.mlp.children()):
            if isinstance(m, torch.nn.Linear):
                codes, scale = quantize_per_token_int8(m.weight.detach())
                m.weight.data = (codes.double() * scale.double()[:, None]).to(dtype)
    return model


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_int8_projections_track_the_model(cuda_device, dtype):
    """Against the same model with dequantised weights: what is left is the activations' quantisation. A row of k values
    of which amax is at most about 4 to 5 times the rms loses amax / 127 / sqrt(12) an element, about 1.2 % of the rms; with
    seven projections in each of two layers, and through their nonlinearities, under ten times that."""
    from tilemix_b200.linear.int8_linear import Int8Linear
    from tilemix_b200.models.int8_projections import quantize_projections_int8

    ids = _ids(cuda_device, 2, 50, seed=4)
    with torch.no_grad():
        ref = _dequantised(_model(cuda_device).to(dtype), dtype)(ids).logits
        model = quantize_projections_int8(_model(cuda_device).to(dtype))
        got = model(ids).logits
    assert sum(isinstance(m, Int8Linear) for m in model.modules()) == 14
    assert 0 < _rel(got, ref) < 0.12
    with pytest.raises(ValueError, match="Int8Linear"):
        quantize_projections_int8(model)


def test_int8_projections_refuse_the_cpu():
    from tilemix_b200.models.int8_projections import quantize_projections_int8

    with pytest.raises(RuntimeError, match="GPU"):
        quantize_projections_int8(_model("cpu"))


def test_int8_projections_are_not_sharded(cuda_device):
    from tilemix_b200.models.int8_projections import quantize_projections_int8
    from tilemix_b200.models.tensor_parallel import shard_model_for_tensor_parallel

    model = quantize_projections_int8(_model(cuda_device))
    with pytest.raises(ValueError, match="cannot be sharded"):
        shard_model_for_tensor_parallel(model, 0, 2)


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_the_whole_path_together(cuda_device, kind):
    """8-bit projections, TileMix prefill (its CUDA norms, rotary and SiLU for Llama), decode over the 4-bit cache: close
    to the fp16 model, and the same again."""
    from tilemix_b200.models.int8_projections import quantize_projections_int8
    from tilemix_b200.models.kv4_cache import Kv4Cache
    from tilemix_b200.models.tilemix_llama import prepare_llama_prefill

    plain = _model(cuda_device, kind, head_dim=128)
    model = _inject(_model(cuda_device, kind, head_dim=128), kind)
    if kind == "llama":
        prepare_llama_prefill(model)
    quantize_projections_int8(model)
    outs = []
    for _ in range(2):
        cache, ref_cache, logits = Kv4Cache(700), None, []
        with torch.no_grad():
            for i, t in enumerate((600, 1, 1, 4)):
                ids = _ids(cuda_device, 2, t, seed=20 + i)
                ref = plain(ids, past_key_values=ref_cache, use_cache=True)
                ref_cache = ref.past_key_values
                logits.append(model(ids, past_key_values=cache, use_cache=True).logits[:, -1])
                # 8-bit activations and weights (above) and 4-bit keys and values: 1/15 of a group's range / sqrt(12)
                # is under 10 % of the rms of normal values, averaged over the keys that a row attends to
                assert _rel(logits[-1], ref.logits[:, -1]) < 0.3
        outs.append(torch.cat(logits))
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_attention_is_injected_before_the_projections_are_quantised(cuda_device, kind):
    """The other way round is refused and leaves the model as it was: the weights to copy are no longer there."""
    from tilemix_b200.models.int8_projections import quantize_projections_int8

    model = quantize_projections_int8(_model(cuda_device, kind))
    before = [layer.self_attn for layer in model.model.layers]
    with pytest.raises(ValueError, match="inject TileMix attention before"):
        _inject(model, kind)
    assert all(layer.self_attn is a for layer, a in zip(model.model.layers, before))


def test_a_cache_filled_in_inference_mode_is_reset_outside_it(cuda_device):
    from tilemix_b200.models.kv4_cache import Kv4Cache

    model = _inject(_model(cuda_device))
    cache, ids = Kv4Cache(64, page_size=16), _ids(cuda_device, 2, 20, seed=3)
    with torch.inference_mode():
        first = model(ids, past_key_values=cache, use_cache=True).logits
        model(ids[:, :2], past_key_values=cache, use_cache=True)
    cache.reset()
    with torch.no_grad():
        again = model(ids, past_key_values=cache, use_cache=True).logits
    assert torch.equal(first, again)
