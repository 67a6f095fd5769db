"""The fast-policy example on a small teacher: its layers are the products of
their quantised parts, its moves the sampler's on its logits, and the engine's
own logits can be sampled where they lie."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fitted(engine):
    import fast_policy

    desc = engine.NetDesc(5, 1, 2, 32, 32, 0)
    params, buffers = engine.synth_network(desc, 3)
    x = engine.synth_positions(desc, 4, 600)
    with engine.CudaInference(desc, params, buffers, 64, 0, engine.TF32X3) as teacher:
        yield desc, teacher, x, fast_policy.FastPolicy.fit(teacher, x, hidden=200)


def test_logits_are_the_layers_products(fitted):
    import azb_ops as A
    import torch

    desc, _, x, policy = fitted
    h = torch.as_tensor(x.reshape(600, -1), device="cuda")
    logits = policy.logits(h)
    for i, (w, b) in enumerate(policy.layers):
        y = A.mx4_values(A.mx4_quantise(h)).double() @ A.mx4_values(w).double().t() + b.double()
        h = y.clamp(min=0).bfloat16() if i < 2 else y
    assert logits.shape == (600, desc.actions)
    # a hidden value may round to the other bfloat16 neighbour, and from there
    # to the other 4-bit neighbour: rarely, and then by one step of a block
    assert (logits.double() - h).abs().median() <= 1e-5 * h.abs().max()


def test_play_draws_legal_moves(fitted):
    import azb_ops as A
    import torch

    desc, _, x, policy = fitted
    h = torch.as_tensor(x.reshape(600, -1), device="cuda")
    legal = torch.rand(600, desc.actions, device="cuda") < 0.4
    legal[:, -1] = True
    noise = torch.rand(600, desc.actions, device="cuda")
    moves, logprob = policy.play(h, noise, legal, temperature=0.9, top_k=10)
    assert bool((moves >= 0).all())
    assert bool(legal.gather(1, moves.clamp(min=0)[:, None]).all()) and bool((logprob <= 0).all())
    again, _ = A.sample_moves(policy.logits(h), noise, legal=legal, temperature=0.9, top_k=10)
    assert torch.equal(moves, again)


def test_it_follows_its_teacher(fitted):
    import torch

    desc, teacher, x, policy = fitted
    ours = policy.logits(torch.as_tensor(x.reshape(600, -1), device="cuda")).cpu().numpy()
    theirs = np.concatenate([teacher.infer(x[i:i + 50])[0] for i in range(0, 600, 50)])
    assert np.corrcoef(ours.ravel(), theirs.ravel())[0, 1] > 0.5


def test_the_engines_logits_sampled_in_place(fitted, engine):
    """azb_infer_device_logits: the sampler on the engine's own stream."""
    import ctypes as C
    import torch

    desc, teacher, x, _ = fitted
    logits = teacher.infer(x[:40])[0]
    noise = torch.rand(40, desc.actions, device="cuda")
    moves = torch.zeros(40, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    a = engine.SampleArgs(logits=teacher.device_logits(), rows=40, cols=desc.actions, ld=desc.actions,
                          noise=noise.data_ptr(), noise_ld=desc.actions, temperature=1.0, top_p=1.0,
                          moves=moves.data_ptr())
    e = C.create_string_buffer(1024)
    teacher.stage(x[:40])
    teacher.enqueue(40)
    assert engine.lib().azb_sample_moves(0, C.byref(a), teacher.stream(), e, 1024) == 0, e.value
    teacher.sync()
    import azb_ops as A

    ref, _ = A.sample_moves(torch.as_tensor(logits, device="cuda"), noise)
    assert torch.equal(moves, ref)


def test_every_logit_is_its_layers_product(fitted):
    """Each layer against 64 bits on the layer's own input, so that no rounding
    of the one before carries over: an fp32 sum of K exact terms, the bias and
    the output's rounding (bfloat16's half a unit is 2^-8 of the value)."""
    import azb_ops as A
    import torch

    desc, _, x, policy = fitted
    h = torch.as_tensor(x.reshape(600, -1), device="cuda")
    logits = policy.logits(h)
    for i, (w, b) in enumerate(policy.layers):
        xq, wq = A.mx4_values(A.mx4_quantise(h)).double(), A.mx4_values(w).double()
        y, size = xq @ wq.t() + b.double(), xq.abs() @ wq.abs().t() + b.double().abs()
        y = y.clamp(min=0) if i < 2 else y
        out = A.mx4_product(h, w, bias=b, relu=i < 2, dtype=torch.bfloat16 if i < 2 else torch.float32)
        tol = (h.shape[1] + 1) * 2.0 ** -23 * size + (2.0 ** -8 if i < 2 else 2.0 ** -24) * y.abs() + 2.0 ** -133
        assert bool(((out.double() - y).abs() <= tol * (1 + 2.0 ** -8)).all())
        h = out
    assert torch.equal(logits, h)
