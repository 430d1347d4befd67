"""FixationReader: the three operators together, from sampled fixations to gradients and to serving steps."""
import math

import pytest
import torch

from fovi_amd.sensing.coords import SamplingCoords


def _reference(reader, x, states, positions, x_positions, lengths):
    """The block in float64 from its parameters."""
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in reader.named_parameters()}
    x, states = (t.detach().double().cpu().requires_grad_(True) for t in (x, states))

    def norm(t, name):
        m = t.mean(-1, keepdim=True)
        h = (t - m) / ((t - m).square().mean(-1, keepdim=True) + 1e-5).sqrt()
        return h * p[name + ".weight"] + p[name + ".bias"]

    def turn(t, pos):
        freqs, at = reader.rotary.freqs.double().cpu(), 0
        angle = []
        for a, n in enumerate(reader.rotary.sections):
            angle.append(pos.double().cpu()[..., a:a + 1] * freqs[at:at + n])
            at += n
        angle = torch.cat(angle, -1)[..., :, None, :]
        u, v, rest = t[..., :at], t[..., at:2 * at], t[..., 2 * at:]
        return torch.cat([u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin(), rest], -1)

    b, n, _ = x.shape
    h, hk, d = reader.heads, reader.kv_heads, reader.head_dim
    kv = (norm(states, "state_norm") @ p["to_kv.weight"].t()).view(b, -1, 2, hk, d)
    k, v = turn(kv[:, :, 0], positions), kv[:, :, 1]
    q = turn((norm(x, "norm") @ p["to_q.weight"].t()).view(b, n, h, d), x_positions)
    k, v = (t.repeat_interleave(h // hk, 2).transpose(1, 2) for t in (k, v))
    s = q.transpose(1, 2) @ k.transpose(2, 3) / d ** 0.5
    s = s.masked_fill(torch.arange(s.shape[-1]) >= lengths.cpu()[:, None, None, None], -float("inf"))
    read = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(b, n, h * d)
    return x + read @ p["to_out.weight"].t() + p["to_out.bias"], x, states, p


def test_positions_of_fixations():
    from fovi_amd.arch.reader import fixation_positions
    coords = SamplingCoords(16, 2.78, 8, style="logpolar")
    pos = fixation_positions(coords, 3, first=2, device="cpu")
    rc = torch.as_tensor(coords.cartesian_rowcol).float()
    n = rc.shape[0]
    assert pos.shape == (3 * n, 3)
    assert pos[:, 0].tolist() == [2.0] * n + [3.0] * n + [4.0] * n
    assert torch.equal(pos[n:2 * n, 1:], rc)


@pytest.mark.gpu
def test_training_step_against_float64():
    """fp32 library products of the projections (2^-24 each) and the operators' 1e-5: 3e-5."""
    from fovi_amd.arch.reader import FixationReader, fixation_positions
    torch.manual_seed(0)
    reader = FixationReader(48, 40, heads=4, head_dim=32, kv_heads=2)
    coords = SamplingCoords(16, 2.78, 8, style="logpolar")
    pos = fixation_positions(coords, 2)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 7, 48, generator=g).cuda().requires_grad_(True)
    states = torch.randn(3, len(pos), 40, generator=g).cuda().requires_grad_(True)
    lengths = torch.tensor([len(pos), 64, 1], device="cuda")
    xpos = torch.cat([torch.full((7, 1), 2.0), torch.zeros(7, 2)], 1).cuda()
    y = reader(x, states, pos, x_positions=xpos, kv_lengths=lengths)
    dy = torch.randn(y.shape, generator=g)
    grads = torch.autograd.grad(y, [x, states] + list(reader.parameters()), dy.cuda())
    ref, rx, rs, p = _reference(reader, x, states, pos, xpos, lengths)
    want = torch.autograd.grad(ref, [rx, rs] + list(p.values()), dy.double())
    for a, b in zip([y] + list(grads), [ref] + list(want)):
        assert ((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm()).item() < 3e-5


@pytest.mark.gpu
def test_serving_reads_what_training_reads():
    """Foveated views through the patch embedding; keys and values of each fixation projected once
    into buffers; a query token reads them with the number of states so far. Equal to the block on
    the states in one piece, up to bf16 roundings of other product shapes (library products)."""
    from fovi_amd.arch.knnvit import KNNPatchEmbedding
    from fovi_amd.arch.reader import FixationReader, fixation_positions
    from fovi_amd.sensing.retina import RetinalTransform
    torch.manual_seed(3)
    retina = RetinalTransform(32, start_res=64, fov=16, cmf_a=2.78, style="logpolar", sampler="grid_bilinear",
                              device="cuda", auto_match_cart_resources=0).eval()
    embed = KNNPatchEmbedding(3, 96, 32, 16, 2.78, style="logpolar", auto_match_cart_resources=0, cart_patch_size=8,
                              patch_overlap_factor=2, new_parameterization=True, sample_cortex=True,
                              ref_frame_side_length=8, device="cuda", bias=True)
    reader = FixationReader(64, 96, heads=2, head_dim=64)
    img = torch.rand(2, 3, 64, 64).cuda()
    n, fixations = embed.out_coords.shape[0], 3
    pos = fixation_positions(embed.out_coords, fixations)
    keys = torch.empty(2, fixations * n, 2, 64, device="cuda", dtype=torch.bfloat16)
    values, x, states = torch.empty_like(keys), torch.randn(2, 1, 64).cuda(), []
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        for f in range(fixations):
            states.append(embed(retina(img, torch.rand(2, 2) * 0.5 + 0.25)))
            at = slice(f * n, (f + 1) * n)
            keys[:, at], values[:, at] = reader.project(states[-1], pos[at])
            lengths = torch.full((2,), (f + 1) * n, device="cuda", dtype=torch.int32)
            y = reader(x, keys=keys, values=values, kv_lengths=lengths)
            want = reader(x, torch.cat(states, 1), pos[:(f + 1) * n])
            assert ((y - want).norm() / (want - x).norm()).item() < 2e-2


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.reader import FixationReader
    reader = FixationReader(16, 16, heads=2, head_dim=16)
    x = torch.zeros(1, 2, 16, device="cuda")
    for kw in ({}, dict(states=x), dict(keys=x), dict(states=x, keys=x, values=x)):
        with pytest.raises(ValueError):
            reader(x, **kw)
    with pytest.raises(ValueError):
        FixationReader(16, 16, heads=3, kv_heads=2)


def test_every_pair_tells_fixations_apart():
    """Fixations are numbered 0, 1, 2, ...: no pair of that axis turns by whole turns between two of the first 20
    (in fp64; the nearest pair of angles is more than 1e-3 of a turn from one another)."""
    from fovi_amd.arch.reader import FixationReader
    for head_dim in (32, 64, 128):
        rope = FixationReader(16, 16, heads=2, head_dim=head_dim, device="cpu").rotary
        turns = torch.arange(20).double()[:, None] * rope.freqs[:rope.sections[0]].double() / (2 * math.pi)
        apart = (turns[:, None] - turns[None] + 0.5) % 1 - 0.5
        assert (apart.abs() + torch.eye(20)[..., None]).min() > 1e-3
    # row and column stay in [-1, 1]: two pi, as the default of the two-axis positions
    assert rope.freqs[rope.sections[0]] == torch.tensor(2 * math.pi)
    same = FixationReader(16, 16, heads=2, scale=2 * math.pi, device="cpu").rotary.freqs
    assert same[0] == torch.tensor(2 * math.pi)
    two = FixationReader(16, 16, heads=2, head_dim=32, sections=(8, 8), device="cpu").rotary
    assert two.freqs[0] == two.freqs[8] == torch.tensor(2 * math.pi)


@pytest.mark.gpu
@pytest.mark.parametrize("create_graph", [False, True])
def test_checkpointed_block(create_graph):
    """Recomputed in the backward, also where the gradients are recorded: each kept tensor is asked for once."""
    from torch.utils.checkpoint import checkpoint
    from fovi_amd.arch.reader import FixationReader
    torch.manual_seed(4)
    reader = FixationReader(32, 24, heads=2, head_dim=16)
    x, states = torch.randn(2, 5, 32, device="cuda"), torch.randn(2, 40, 24, device="cuda")
    pos, xpos = torch.rand(40, 3, device="cuda"), torch.rand(5, 3, device="cuda")
    x.requires_grad_(True)

    def block(x):
        return reader(x, states, pos, x_positions=xpos)

    want = torch.autograd.grad(block(x).square().sum(), [x] + list(reader.parameters()))
    y = checkpoint(block, x, use_reentrant=False)
    got = torch.autograd.grad(y.square().sum(), [x] + list(reader.parameters()), create_graph=create_graph)
    for a, b in zip(got, want):
        assert ((a - b).norm() / b.norm()).item() < 1e-6
