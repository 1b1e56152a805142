"""The mel producer (tts_amd/acoustic.py) against an independent numpy forward pass written in
Keras conventions (weight layouts, gate order, masking, epsilon) of the reference model
TTS/Fastspeech_1.py:95-128.  TensorFlow is not available and the reference ships no weights, so
equality with the Keras model itself is unpinned; this pins the layout mapping and the
reference's call-graph quirks."""
import numpy as np
import pytest
import torch

from tts_amd.acoustic import FastSpeechAcousticModel, length_regulate

VOCAB = 72  # TTS/train.py:43


def _sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def keras_lstm(x, mask, kernel, recurrent, bias, go_backwards=False):
    """LSTM(return_sequences=True) on one row; masked steps carry the state and repeat the output."""
    units = recurrent.shape[0]
    steps = range(len(x) - 1, -1, -1) if go_backwards else range(len(x))
    h = np.zeros(units)
    c = np.zeros(units)
    prev_out = np.zeros(units)
    out = np.zeros((len(x), units))
    for t in steps:
        if mask[t]:
            z = x[t] @ kernel + h @ recurrent + bias
            i, f, g, o = np.split(z, 4)
            c = _sigmoid(f) * c + _sigmoid(i) * np.tanh(g)
            h = _sigmoid(o) * np.tanh(c)
            prev_out = h
        out[t] = prev_out
    return out


def keras_conv1d(x, kernel, bias, dilation=1):
    """Conv1D(padding='same'): kernel (k, in, out); x (T, in)."""
    k = kernel.shape[0]
    total = dilation * (k - 1)
    left = total // 2
    xp = np.pad(x, ((left, total - left), (0, 0)))
    out = np.zeros((len(x), kernel.shape[2]))
    for j in range(k):
        out += xp[j * dilation: j * dilation + len(x)] @ kernel[j]
    return out + bias


def layer_norm(x, gamma, beta):
    mu = x.mean(-1, keepdims=True)
    var = x.var(-1, keepdims=True)
    return (x - mu) / np.sqrt(var + 1e-3) * gamma + beta


def random_weights(rng, mel_dim=80, hidden=256, emb=256):
    w = {"embed": rng.normal(0, 0.5, (VOCAB, emb))}
    dims = [(emb, 512), (1024, 512), (1024, 128)]
    for n, (i, u) in enumerate(dims, 1):
        for d in ("fwd", "bwd"):
            w[f"lstm{n}_{d}_kernel"] = rng.normal(0, 1 / np.sqrt(i), (i, 4 * u))
            w[f"lstm{n}_{d}_recurrent"] = rng.normal(0, 1 / np.sqrt(u), (u, 4 * u))
            w[f"lstm{n}_{d}_bias"] = rng.normal(0, 0.1, 4 * u)
    for n, i in ((1, 256), (2, hidden)):
        w[f"enc_conv{n}_kernel"] = rng.normal(0, 1 / np.sqrt(5 * i), (5, i, hidden))
        w[f"enc_conv{n}_bias"] = rng.normal(0, 0.1, hidden)
        w[f"enc_norm{n}_gamma"] = rng.normal(1, 0.1, hidden)
        w[f"enc_norm{n}_beta"] = rng.normal(0, 0.1, hidden)
    for n in (1, 2, 3):
        w[f"dur_conv{n}_kernel"] = rng.normal(0, 1 / np.sqrt(3 * hidden), (3, hidden, hidden))
        w[f"dur_conv{n}_bias"] = rng.normal(0, 0.1, hidden)
        w[f"dur_norm{n}_gamma"] = rng.normal(1, 0.1, hidden)
        w[f"dur_norm{n}_beta"] = rng.normal(0, 0.1, hidden)
    w["dur_out_kernel"] = rng.normal(0, 0.1, (hidden, 1))
    w["dur_out_bias"] = rng.normal(0, 0.1, 1)
    w["mel_out_kernel"] = rng.normal(0, 1 / np.sqrt(hidden), (1, hidden, mel_dim))
    w["mel_out_bias"] = rng.normal(0, 0.1, mel_dim)
    w["post_conv_kernel"] = rng.normal(0, 1 / np.sqrt(5 * mel_dim), (5, mel_dim, mel_dim))
    w["post_conv_bias"] = rng.normal(0, 0.1, mel_dim)
    w["post_bn_gamma"] = rng.normal(1, 0.1, mel_dim)
    w["post_bn_beta"] = rng.normal(0, 0.1, mel_dim)
    w["post_bn_mean"] = rng.normal(0, 0.1, mel_dim)
    w["post_bn_var"] = rng.uniform(0.5, 1.5, mel_dim)
    # the module stores float32 parameters: use values float32 holds exactly
    return {k: v.astype(np.float32).astype(np.float64) for k, v in w.items()}


def numpy_forward(w, ids, durations):
    """Row 0 through the reference's call graph (TTS/Fastspeech_1.py:113-128)."""
    mask = ids != 0
    x = w["embed"][ids]
    for n in (1, 2, 3):
        f = keras_lstm(x, mask, w[f"lstm{n}_fwd_kernel"], w[f"lstm{n}_fwd_recurrent"], w[f"lstm{n}_fwd_bias"])
        b = keras_lstm(x, mask, w[f"lstm{n}_bwd_kernel"], w[f"lstm{n}_bwd_recurrent"], w[f"lstm{n}_bwd_bias"],
                       go_backwards=True)
        x = np.concatenate([f, b], axis=-1)
    for n in (1, 2):
        x = np.maximum(keras_conv1d(x, w[f"enc_conv{n}_kernel"], w[f"enc_conv{n}_bias"], dilation=2), 0)
        x = layer_norm(x, w[f"enc_norm{n}_gamma"], w[f"enc_norm{n}_beta"])
    dur = x
    for n in (1, 2, 3):
        dur = np.maximum(keras_conv1d(dur, w[f"dur_conv{n}_kernel"], w[f"dur_conv{n}_bias"]), 0)
        dur = layer_norm(dur, w[f"dur_norm{n}_gamma"], w[f"dur_norm{n}_beta"])
    dur = dur @ w["dur_out_kernel"] + w["dur_out_bias"]
    d = np.round(np.exp(durations)).astype(np.int64)
    reps = np.repeat(np.arange(len(ids)), d)
    x = np.repeat(x, d, axis=0)[reps]
    mel = keras_conv1d(x, w["mel_out_kernel"], w["mel_out_bias"])
    post = mel
    for i in range(5):
        post = np.tanh(keras_conv1d(post, w["post_conv_kernel"], w["post_conv_bias"]))
        if i < 4:
            post = (post - w["post_bn_mean"]) / np.sqrt(w["post_bn_var"] + 1e-3) * w["post_bn_gamma"] + w["post_bn_beta"]
    return mel + post, dur


@pytest.mark.parametrize("pad", [0, 4])
def test_matches_keras_convention_forward(pad):
    rng = np.random.default_rng(5)
    w = random_weights(rng)
    n = 9
    ids = np.concatenate([rng.integers(1, VOCAB, n), np.zeros(pad, np.int64)])
    durations = np.log(np.concatenate([rng.integers(1, 6, n), np.ones(pad)]).astype(np.float64))
    model = FastSpeechAcousticModel(VOCAB).load_keras_weights(w).double()
    out = model((ids[None], durations[None]))
    want, want_dur = numpy_forward(w, ids, durations)
    assert out.shape == (1, want.shape[0], 80)
    assert np.abs(out[0].numpy() - want).max() < 1e-9
    assert np.abs(model.last_duration_prediction[0].numpy() - want_dur).max() < 1e-9


def test_length_regulator_double_index():
    # durations 2, 1, 3 -> frame owner p = [0,0,1,2,2,2]; the reference gathers the expanded
    # sequence with p again: out[i] = expanded[p[i]] = x[p[p[i]]] = x[[0,0,0,1,1,1]]
    x = torch.arange(3, dtype=torch.float32)[None, :, None]
    out = length_regulate(x, torch.log(torch.tensor([[2.0, 1.0, 3.0]])))
    assert out[0, :, 0].tolist() == [0, 0, 0, 1, 1, 1]


def test_rejects_inner_padding_and_shape_mismatch():
    model = FastSpeechAcousticModel(VOCAB)
    with pytest.raises(ValueError):
        model((np.array([[3, 0, 5]]), np.zeros((1, 3))))
    with pytest.raises(ValueError):
        model((np.array([[3, 4, 5]]), np.zeros((1, 4))))
    # zero frames for a phoneme can make tf.gather's index run past the expanded sequence
    with pytest.raises(IndexError):
        model((np.array([[3, 4, 5]]), np.log(np.array([[0.4, 0.4, 1.0]]))))


def test_float32_close_to_float64():
    rng = np.random.default_rng(6)
    w = random_weights(rng)
    ids = rng.integers(1, VOCAB, 12)
    durations = np.log(rng.integers(2, 7, 12).astype(np.float64))
    m32 = FastSpeechAcousticModel(VOCAB).load_keras_weights(w)
    out = m32((ids[None], durations[None].astype(np.float32)))[0].numpy()
    want, _ = numpy_forward(w, ids, durations)
    assert np.linalg.norm(out - want) / np.linalg.norm(want) < 1e-4


def test_mxfp4_needs_a_gpu_and_leaves_the_state_dict_alone():
    model = FastSpeechAcousticModel(VOCAB)
    keys = list(model.state_dict())
    assert not any("mxfp4" in k for k in keys) and "encoder.block1.conv.weight" in keys and "mel_out.weight" in keys
    with pytest.raises(ValueError, match="ROCm GPU"):
        model.use_mxfp4()
    assert model.use_mxfp4(False) is model


def quantised(weights):
    return FastSpeechAcousticModel(VOCAB).load_keras_weights(weights).cuda().use_mxfp4()


def same_layers(model, other):
    pairs = list(zip(model._mxfp4_layers(), other._mxfp4_layers(), strict=True))
    return all(torch.equal(a.mxfp4_data, b.mxfp4_data) for a, b in pairs)


@pytest.mark.gpu
def test_mxfp4_blocks_against_the_oracle_and_back():
    from oracle import blocks_oracle as O
    rng = np.random.default_rng(7)
    w = random_weights(rng)
    ids = np.concatenate([rng.integers(1, VOCAB, 40), np.zeros(3, np.int64)])[None]
    durations = np.log(rng.integers(1, 6, ids.shape).astype(np.float64)).astype(np.float32)
    model = FastSpeechAcousticModel(VOCAB).load_keras_weights(w).cuda()
    plain = model((ids, durations))
    keys = list(model.state_dict())
    assert model.use_mxfp4() is model and list(model.state_dict()) == keys
    seen = []
    blocks = [model.encoder.block1, model.encoder.block2, *model.duration_predictor.blocks]
    hooks = [b.register_forward_hook(lambda m, args, out: seen.append((m, args[0], out))) for b in blocks]
    mel = model((ids, durations))
    for h in hooks:
        h.remove()
    assert [s[0] for s in seen] == blocks
    # each block on the input that it was given, so that roundings upstream are no errors here
    for block, x, out in seen:
        conv, norm = block.conv, block.norm
        d = [v.detach().cpu().double().numpy() for v in (x, conv.weight.permute(0, 2, 1), conv.bias, norm.weight, norm.bias, out)]
        y, size = O.conv1d(O.mxfp4_round(d[0]), O.mxfp4_round(d[1]), d[2], conv.dilation[0])
        y = np.maximum(y, 0)
        want = O.norm(y, "layer", d[3], d[4], 1e-3)
        k = conv.weight.shape[1] * conv.weight.shape[2]
        # the product's float sum (k + 1 steps of at most 2^-23 of the magnitudes), then the norm: an error of
        # the row reaches an element directly and through mean and variance; its own sums are short
        worst = ((k + 1) * 2.0 ** -23 * size).max(-1, keepdims=True) + 100 * 2.0 ** -24 * np.abs(y).mean(-1, keepdims=True)
        centred = y - y.mean(-1, keepdims=True)
        r = 1 / np.sqrt((centred ** 2).mean(-1, keepdims=True) + 1e-3)
        hat = np.abs(centred) * r
        bound = np.abs(d[3]) * (r * worst * (2 + hat) + 120 * 2.0 ** -24 * (hat + r * np.abs(y))) + 8 * 2.0 ** -24 * (
            np.abs(want) + np.abs(d[4]))
        assert (np.abs(d[5] - want) <= bound).all()
    assert mel.shape == plain.shape and torch.isfinite(mel).all() and not torch.equal(mel, plain)
    # loading weights quantises them anew
    other = random_weights(np.random.default_rng(8))
    assert same_layers(model.load_keras_weights(other), quantised(other))
    model.load_state_dict(FastSpeechAcousticModel(VOCAB).load_keras_weights(w).state_dict())
    assert same_layers(model, quantised(w)) and not same_layers(model, quantised(other))
    model.use_mxfp4(False)
    assert all(layer.mxfp4_data is None for layer in model._mxfp4_layers())
    # float32 is within 1e-4 of float64 (above), so two runs of it are within twice that of each other: the
    # libraries behind it may choose another algorithm from call to call
    assert (model((ids, durations)) - plain).norm() < 2e-4 * plain.norm()


@pytest.mark.gpu
def test_mxfp4_follows_the_weights_of_a_part_and_of_a_copy():
    import copy
    w, other = random_weights(np.random.default_rng(11)), random_weights(np.random.default_rng(12))
    model = quantised(w)
    want = FastSpeechAcousticModel(VOCAB).load_keras_weights(other)
    twin = copy.deepcopy(model)
    for name, part in want.named_children():
        getattr(model, name).load_state_dict(part.state_dict())
    assert same_layers(model, quantised(other)) and same_layers(twin, quantised(w))
    torch.nn.ModuleList([twin]).load_state_dict({"0." + k: v for k, v in want.state_dict().items()})
    assert same_layers(twin, model)


@pytest.mark.gpu
def test_mxfp4_model_feeds_the_vocoder():
    from tts_amd.acoustic import synthesize
    rng = np.random.default_rng(9)
    model = FastSpeechAcousticModel(VOCAB).load_keras_weights(random_weights(rng)).cuda().use_mxfp4()
    ids = rng.integers(1, VOCAB, 30)[None]
    durations = np.log(rng.integers(2, 5, ids.shape).astype(np.float64)).astype(np.float32)
    audio, mel = synthesize(model, ids, durations, -61.6, 20.4, return_mel=True, n_iter=4, init_phase=1)
    assert torch.isfinite(audio).all() and audio.shape == (256 * (mel.shape[0] - 1),)


def held_in_mxfp4(model):
    """The state of a model that was moved to the host after use_mxfp4(): its buffers come along."""
    for layer in model._mxfp4_layers():
        n, c, taps = layer.weight.shape
        layer.mxfp4_data = torch.zeros(n * taps * -(-c // 128) * 68, dtype=torch.uint8)
    return model


@pytest.mark.parametrize("how", ["state_dict", "keras", "assign"])
def test_mxfp4_model_on_the_host_loads_weights_whole(how):
    w = random_weights(np.random.default_rng(13))
    model, want = held_in_mxfp4(FastSpeechAcousticModel(VOCAB)), FastSpeechAcousticModel(VOCAB).load_keras_weights(w)
    if how == "keras":
        model.load_keras_weights(w)
    else:
        model.load_state_dict(want.state_dict(), assign=how == "assign")
    got = model.state_dict()
    assert all(torch.equal(got[k], v) for k, v in want.state_dict().items())
    assert all(layer.stale for layer in model._mxfp4_layers())
    # what was quantised before does not stand for these weights
    with pytest.raises(ValueError, match="cannot be quantised"):
        model((np.array([[3, 4]]), np.zeros((1, 2), np.float32)))
    assert all(layer.stale for layer in model.float()._mxfp4_layers())
    inputs = np.array([[3, 4, 5]]), np.ones((1, 3), np.float32)
    assert torch.equal(model.use_mxfp4(False)(inputs), want(inputs))


@pytest.mark.gpu
def test_mxfp4_weights_loaded_on_the_host_or_in_another_type_are_quantised_on_the_way_back():
    w, other = random_weights(np.random.default_rng(14)), random_weights(np.random.default_rng(15))
    state = FastSpeechAcousticModel(VOCAB).load_keras_weights(other).state_dict()
    for there, back in (("cpu", "cuda"), (torch.float64, torch.float32)):
        model = quantised(w).to(there)
        model.load_state_dict(state)
        assert all(layer.stale for layer in model._mxfp4_layers())
        assert same_layers(model.to(back), quantised(other)) and not any(layer.stale for layer in model._mxfp4_layers())


def test_mxfp4_weights_are_quantised_anew_in_place(monkeypatch):
    from types import SimpleNamespace
    from tts_amd import acoustic
    made = iter((1, 2))
    monkeypatch.setattr(acoustic, "mxfp4_quantize", lambda w: SimpleNamespace(data=torch.full((68,), next(made), dtype=torch.uint8)))
    layer = FastSpeechAcousticModel(VOCAB).mel_out
    layer.quantize(True)
    kept = layer.mxfp4_data
    layer.quantize(True)
    assert layer.mxfp4_data is kept and (kept == 2).all()


@pytest.mark.gpu
def test_mxfp4_graph_follows_the_weights():
    w, other = random_weights(np.random.default_rng(16)), random_weights(np.random.default_rng(17))
    model, want = quantised(w), quantised(other)
    blocks = [(m.encoder.block1, m.duration_predictor.blocks[0]) for m in (model, want)]
    x = torch.randn(2, 30, 256, device="cuda")
    with torch.no_grad():
        [b(x) for b in blocks[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [b(x) for b in blocks[0]]
        for load in (lambda: None, lambda: model.load_keras_weights(other), lambda: model.load_keras_weights(w),
                     lambda: model.load_state_dict(want.state_dict())):
            load()
            eager = [b(x) for b in blocks[0]]
            for out in outs:
                out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        assert all(torch.equal(a, b(x)) for a, b in zip(outs, blocks[1]))


def test_mxfp4_copy_does_not_outlive_a_keras_load_that_ends_early():
    w = random_weights(np.random.default_rng(18))
    model = held_in_mxfp4(FastSpeechAcousticModel(VOCAB))
    del w["post_bn_var"]
    with pytest.raises(KeyError):
        model.load_keras_weights(w)
    assert np.array_equal(model.mel_out.bias.detach().numpy(), w["mel_out_bias"])
    assert all(layer.stale for layer in model._mxfp4_layers())


def test_convolutions_can_be_replaced():
    """A layer of another kind, of one's own or of a library, in the place of one of the model's."""
    model = FastSpeechAcousticModel(VOCAB).load_keras_weights(random_weights(np.random.default_rng(19)))
    inputs = np.array([[3, 4, 5]]), np.ones((1, 3), np.float32)
    want = model(inputs)

    def plain(conv):
        other = torch.nn.Conv1d(conv.in_channels, conv.out_channels, conv.kernel_size, padding="same", dilation=conv.dilation)
        other.load_state_dict(conv.state_dict())
        return other

    model.mel_out, model.encoder.block2.conv = plain(model.mel_out), plain(model.encoder.block2.conv)
    assert torch.equal(model(inputs), want)


def through(model, modules, run):
    """What forward hooks on the modules see while `run` runs."""
    seen = {}
    hooks = [m.register_forward_hook(lambda m, args, out: seen.__setitem__(m, (args[0], out))) for m in modules]
    out = run()
    for h in hooks:
        h.remove()
    return out, [seen.get(m) for m in modules]


def test_hooks_on_convolutions_fire_in_mxfp4(monkeypatch):
    from tts_amd import acoustic

    def product(x, weight, bias, dilation=1, activation=None):
        y = bias + x.sum(-1, keepdim=True) * (-1.0) ** torch.arange(len(bias))
        return torch.relu(y) if activation else y

    for name in ("mxfp4_conv1d", "mxfp4_linear"):
        monkeypatch.setattr(acoustic, name, product)
    monkeypatch.setattr(acoustic, "block_norm", lambda u, post: u)
    model = held_in_mxfp4(FastSpeechAcousticModel(VOCAB))
    inputs = np.array([[3, 4, 5]]), np.ones((1, 3), np.float32)
    want, convs = model(inputs), model._mxfp4_layers()
    out, seen = through(model, convs, lambda: model(inputs))
    assert torch.equal(out, want) and None not in seen
    for conv, (x, y) in zip(convs, seen):
        # (B, C, T), and before the rectifier, as in the float form
        assert torch.equal(y, product(x.transpose(1, 2), None, conv.bias).transpose(1, 2)) and (y < 0).any()


@pytest.mark.gpu
def test_hooks_on_convolutions_change_nothing_in_mxfp4():
    model = quantised(random_weights(np.random.default_rng(20)))
    block, x = model.encoder.block1, torch.randn(2, 30, 256, device="cuda")
    with torch.no_grad():
        want = block(x)
        out, [(given, y)] = through(block, [block.conv], lambda: block(x))
        assert torch.equal(out, want) and torch.equal(given.transpose(1, 2), x) and (y < 0).any()
        assert torch.equal(block.conv(given), y)


def test_norms_are_called_as_modules_with_their_own_eps(monkeypatch):
    from tts_amd import acoustic
    calls = []

    def end(u, post):
        calls.append(post)
        return torch.nn.functional.layer_norm(u, u.shape[-1:], post.weight, post.bias, post.eps)

    monkeypatch.setattr(acoustic, "block_norm", end)
    # without convolutions of a kind that the host cannot run
    monkeypatch.setattr(acoustic._SequenceConv, "quantize", lambda self, on: None)
    model = FastSpeechAcousticModel(VOCAB)
    inputs = np.array([[3, 4, 5]]), np.ones((1, 3), np.float32)
    norms = [model.encoder.block1.norm, model.encoder.block2.norm, *(b.norm for b in model.duration_predictor.blocks)]
    for n, norm in enumerate(norms):
        norm.eps = 1e-3 * 2 ** n
    want, plain = through(model, norms, lambda: model(inputs))
    assert not calls
    got, seen = through(model, norms, lambda: model.use_mxfp4()(inputs))
    assert [c.eps for c in calls] == [norm.eps for norm in norms] and torch.equal(got, want)
    assert all(torch.equal(a[1], b[1]) for a, b in zip(seen, plain))
    model.encoder.block1.norm = torch.nn.Identity()
    model(inputs)
    assert len(calls) == 9
    calls.clear()
    model.use_mxfp4(False)(inputs)
    assert not calls


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_mxfp4_layers_against_the_oracle_before_and_after_a_reload(dtype):
    """Every convolution, norm and the mel head on an input of its own, without the LSTMs of a library between them."""
    import copy
    from oracle import blocks_oracle as O
    from test_blocks import check_block_norm, check_product
    from tts_amd import Norm
    w, other = random_weights(np.random.default_rng(21)), random_weights(np.random.default_rng(22))
    rng = np.random.default_rng(23)

    def check(model, weights):
        layers = {"enc_conv1": model.encoder.block1, "enc_conv2": model.encoder.block2, "mel_out": model.mel_out,
                  **{f"dur_conv{n}": b for n, b in enumerate(model.duration_predictor.blocks, 1)}}
        for name, layer in layers.items():
            conv, norm = (layer, None) if name == "mel_out" else (layer.conv, layer.norm)
            x = torch.from_numpy(rng.normal(0, 1, (2, 21, 256))).to(dtype).cuda()
            xv = O.mxfp4_round(x.cpu().double().numpy())

            def held(key):  # what the layer keeps of a loaded array
                return torch.from_numpy(weights[name + key]).float().to(dtype).double().numpy()

            wv = O.mxfp4_round(held("_kernel").transpose(2, 0, 1))
            want, size = O.conv1d(xv, wv, held("_bias"), conv.dilation[0])
            k = wv.shape[1] * wv.shape[2]
            if norm is None:
                check_product(conv(x.transpose(1, 2)).transpose(1, 2), want, size, k, dtype)
                continue
            out, [(_, y), (u, _)] = through(layer, [conv, norm], lambda: layer(x))
            check_product(y.transpose(1, 2), want, size, k, dtype)
            assert torch.equal(u, torch.relu(y.transpose(1, 2)))
            check_block_norm(u, Norm(norm.weight, norm.bias, norm.eps), None, None, None, None, out)
            assert torch.equal(layer(x), out)  # the rectifier within the product

    with torch.no_grad():
        model = FastSpeechAcousticModel(VOCAB).load_keras_weights(w).cuda().to(dtype).use_mxfp4()
        check(model, w)
        twin = copy.deepcopy(model)
        check(model.load_keras_weights(other), other)
        check(twin, w)
        model.load_state_dict(twin.state_dict())
        check(model, w)
        twin.cpu().load_state_dict(FastSpeechAcousticModel(VOCAB).load_keras_weights(other).state_dict())
        check(twin.cuda(), other)


def test_a_forward_put_in_place_of_the_layers_runs_in_mxfp4():
    model = held_in_mxfp4(FastSpeechAcousticModel(VOCAB))
    for layer in model._mxfp4_layers():
        layer.forward = super(type(layer), layer).forward  # as libraries that place layers on devices wrap it
    inputs = np.array([[3, 4, 5]]), np.ones((1, 3), np.float32)
    got = model(inputs)
    assert torch.equal(got, model.use_mxfp4(False)(inputs))


def test_mxfp4_weights_quantised_in_inference_mode_stay_in_place(monkeypatch):
    from types import SimpleNamespace
    from tts_amd import acoustic
    made = iter((1, 2, 3))
    monkeypatch.setattr(acoustic, "mxfp4_quantize", lambda w: SimpleNamespace(data=torch.full((68,), next(made), dtype=torch.uint8)))
    layer = FastSpeechAcousticModel(VOCAB).mel_out
    with torch.inference_mode():
        layer.quantize(True)
        kept = layer.mxfp4_data
        layer.quantize(True)
        assert layer.mxfp4_data is kept
    layer.quantize(True)
    assert layer.mxfp4_data is kept and (kept == 3).all()
