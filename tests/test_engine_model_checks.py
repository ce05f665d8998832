"""The rollout and the recurrence read a model's parameters by address: a model with another kind of layer in place of one that
they know is refused before anything is launched."""
import copy

import pytest
import torch

from dreamer_amd import _native as N
from dreamer_amd import imagine, mx4, norm, observe
from helpers import DIMS, build_models


def four_bit(linear):
    """The layer in 4 bits (zero codes: only its form matters here)."""
    nb = -(-linear.in_features // 32)
    codes = torch.zeros(linear.out_features, nb * 16, dtype=torch.uint8, device=linear.weight.device)
    scales = torch.full((linear.out_features, nb), 127, dtype=torch.uint8, device=linear.weight.device)
    return mx4.MX4Linear(mx4.MX4Tensor._of(codes, scales, linear.in_features), linear.bias)


def parts(d, wm, actor, critic):
    S = d["D"] + d["L"] * d["K"]
    return {"dyn": (wm.dyn, d["D"]), "rew": (wm.rew, S), "cont": (wm.cont, S), "actor": (actor, S), "critic": (critic, S)}


def test_an_mlp_as_it_is_built_gives_its_addresses():
    d = DIMS["small"]
    for name, (m, width) in parts(d, *build_models(d, 3)).items():
        s = imagine._mlp_struct(m.mlp, m.head, width, name)
        lin = [x for x in m.mlp if isinstance(x, torch.nn.Linear)]
        ln = [x for x in m.mlp if isinstance(x, torch.nn.LayerNorm)]
        assert (s.n_layers, s.in_dim, s.hidden, s.out_dim) == (len(lin), width, d["M"], m.head.out_features)
        assert [s.w[i] for i in range(s.n_layers)] == [x.weight.data_ptr() for x in lin]
        assert [s.b[i] for i in range(s.n_layers)] == [x.bias.data_ptr() for x in lin]
        assert [s.ln_g[i] for i in range(s.n_layers)] == [x.weight.data_ptr() for x in ln]
        assert [s.ln_b[i] for i in range(s.n_layers)] == [x.bias.data_ptr() for x in ln]
        assert (s.head_w, s.head_b) == (m.head.weight.data_ptr(), m.head.bias.data_ptr())


@pytest.mark.parametrize("part", ["dyn", "rew", "cont", "actor", "critic"])
def test_a_4_bit_layer_in_an_mlp_is_refused(part):
    d = DIMS["small"]
    m, width = parts(d, *build_models(d, 3))[part]
    for layer in (0, 3):
        mlp = copy.deepcopy(m.mlp)
        mlp[layer] = four_bit(mlp[layer])
        with pytest.raises(N.NativeError, match=f"{part}: .*MX4Linear"):
            imagine._mlp_struct(mlp, m.head, width, part)
    with pytest.raises(N.NativeError, match=f"{part}: .*MX4Linear"):
        imagine._mlp_struct(m.mlp, four_bit(m.head), width, part)


def test_other_layers_in_an_mlp_are_refused():
    d = DIMS["small"]
    _, actor, _ = build_models(d, 3)
    S, M = d["D"] + d["L"] * d["K"], d["M"]
    changes = {
        "a missing norm": lambda m: m.__delitem__(1), "a missing activation": lambda m: m.__delitem__(5),
        "another activation": lambda m: m.__setitem__(2, torch.nn.ReLU()),
        "a norm without weights": lambda m: m.__setitem__(1, norm.LayerNorm(M, elementwise_affine=False)),
        "a norm without bias": lambda m: m.__setitem__(4, norm.LayerNorm(M, bias=False)),
        "another eps": lambda m: m.__setitem__(1, norm.LayerNorm(M, eps=1e-3)),
        "another width": lambda m: m.__setitem__(3, torch.nn.Linear(M, 2 * M)),
        "another input": lambda m: m.__setitem__(0, torch.nn.Linear(S - 1, M)),
        "no bias": lambda m: m.__setitem__(0, torch.nn.Linear(S, M, bias=False)),
        "a computed weight": lambda m: torch.nn.utils.parametrizations.weight_norm(m[0]),
        "nothing": lambda m: [m.__delitem__(0) for _ in range(6)],
        "too many layers": lambda m: m.extend([copy.deepcopy(x) for _ in range(3) for x in list(m)[3:6]]),
    }
    for what, change in changes.items():
        mlp = copy.deepcopy(actor.mlp)
        change(mlp)
        with pytest.raises(N.NativeError, match="actor: "):
            imagine._mlp_struct(mlp, actor.head, S, "actor")
            pytest.fail(what)
    mlp = copy.deepcopy(actor.mlp)
    mlp[1] = norm.LayerNorm(M)                       # the package's own norm is a nn.LayerNorm in form
    assert imagine._mlp_struct(mlp, actor.head, S, "actor").ln_g[0] == mlp[1].weight.data_ptr()


def test_other_layers_in_the_recurrence_are_refused():
    d = DIMS["small"]
    wm, _, _ = build_models(d, 3)
    observe.check_sequence_model(wm)
    D, L = d["D"], wm.seq.linear
    for name, layer in (("linear", four_bit(L)), ("linear", torch.nn.Linear(L.in_features, D + 4)), ("linear", torch.nn.Linear(L.in_features, D, bias=False)),
                        ("gru", torch.nn.GRUCell(D, 2 * D)), ("gru", torch.nn.GRUCell(D, D, bias=False)), ("gru", torch.nn.LSTMCell(D, D)),
                        ("a_emb", torch.nn.Embedding(d["A"] + 1, 64)), ("a_emb", torch.nn.Embedding(d["A"], 32))):
        other = copy.deepcopy(wm)
        setattr(other.seq, name, layer)
        with pytest.raises(N.NativeError, match="seq"):
            observe.check_sequence_model(other)


@pytest.mark.gpu
def test_the_engines_refuse_such_models_on_the_device():
    from dreamer_amd.world_model import WorldModelState
    from helpers import start_state
    d = DIMS["small"]
    wm, actor, critic = (m.to("cuda:0") for m in build_models(d, 3))
    h0, z0, _ = (t.to("cuda:0") for t in start_state(d, 3))
    start = WorldModelState(h=h0, z=z0)
    good = imagine.imagine(wm, actor, critic, start, d["H"], 0.99, 0.95)
    # a layer that is replaced behind the engine's back: the engine of the first call is still there
    plain = actor.mlp[0]
    actor.mlp[0] = mx4.MX4Linear.from_linear(plain)
    with pytest.raises(N.NativeError, match="actor: .*MX4Linear"):
        imagine.imagine(wm, actor, critic, start, d["H"], 0.99, 0.95)
    with pytest.raises(N.NativeError, match="actor: .*MX4Linear"):
        imagine.ImagineEngine(wm, actor, critic)
    actor(start)                                      # evaluated module by module it acts
    actor.mlp[0] = plain
    lin = wm.seq.linear
    wm.seq.linear = mx4.MX4Linear.from_linear(lin)
    obs = torch.zeros(2, *d["obs_shape"], device="cuda:0")
    with torch.no_grad(), pytest.raises(N.NativeError, match="seq.linear"):
        wm.act_step(WorldModelState(h=h0[:2], z=z0[:2]), torch.zeros(2, dtype=torch.int64, device="cuda:0"), obs)
    with pytest.raises(N.NativeError, match="seq.linear"):
        imagine.imagine(wm, actor, critic, start, d["H"], 0.99, 0.95)
    wm.seq.linear = lin
    assert set(imagine.imagine(wm, actor, critic, start, d["H"], 0.99, 0.95)) == set(good)
