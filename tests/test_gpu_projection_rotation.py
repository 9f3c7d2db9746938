"""The projected pipeline's norm and rotation of Q and K (``qk_rotation``).

Its tiles are the rows that ``normalize_rotate_qk`` gives for the whole call,
so the output equals, bit for bit, that of a projection callback that does the
same; against 64 bits the usual tolerance of the projected pipeline applies
(16-bit projections, attention and output projection one after the other).
"""

from __future__ import annotations

import pytest
import torch

from paged_reference import normalized, rotated
from seqattn import (
    ProjectedAttentionRunner,
    ProjectionPipelineConfig,
    QKRotation,
    StreamingAttentionConfig,
    build_plan,
    rotary_frequencies,
    streaming_projected_self_attention,
)
from seqattn.kernels import normalize_rotate_qk

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, HEADS, KV_HEADS, DIM = 97, 64, 4, 2, 32
SECTIONS = (4, 6, 6)


def parts(seed=3):
    gen = torch.Generator().manual_seed(seed)
    hidden = torch.randn((TOKENS, HIDDEN), generator=gen).to(torch.bfloat16).pin_memory()
    weight = (torch.randn((HIDDEN, (HEADS + 2 * KV_HEADS) * DIM), generator=gen) / HIDDEN**0.5).to(torch.bfloat16)
    t = torch.arange(TOKENS)
    rotation = QKRotation(
        positions=torch.stack([t // 24, t // 6 % 4, t % 6]).cuda(), frequencies=rotary_frequencies(SECTIONS),
        sections=SECTIONS, q_weight=(1 + 0.1 * torch.randn(DIM, generator=gen)).to(torch.bfloat16).cuda(),
        k_weight=(1 + 0.1 * torch.randn(DIM, generator=gen)).cuda(), eps=1e-5,
    )
    return hidden, weight, rotation


def run(residency, hidden, project, rotation, pinned_chunk=31):
    config = StreamingAttentionConfig(backend="hip", q_chunk_tokens=41, kv_chunk_tokens=29)
    plan = build_plan(q_heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, dtype=torch.bfloat16, device="cuda",
                      max_q_tokens=TOKENS, max_kv_tokens=TOKENS, config=config)
    runner = ProjectedAttentionRunner(
        plan, config, ProjectionPipelineConfig(projection_chunk_tokens=pinned_chunk, qkv_residency=residency))
    cu = torch.tensor([0, 40, TOKENS], dtype=torch.int32)
    out = runner(hidden, cu, project_qkv=project, output_projector=lambda tile, start, stop: tile,
                 output_features=HEADS * DIM, causal=True, qk_rotation=rotation)
    torch.cuda.synchronize()
    return runner, out.clone()


@pytest.mark.parametrize("residency", ["host", "hbm"])
def test_rotation_equals_a_callback_that_rotates(residency):
    hidden, weight, rotation = parts()
    w = weight.cuda()

    def project(tile, start, stop):
        return (tile @ w).view(stop - start, HEADS + 2 * KV_HEADS, DIM).split([HEADS, KV_HEADS, KV_HEADS], dim=1)

    def project_and_rotate(tile, start, stop):
        q, k, v = project(tile, start, stop)
        q, k = normalize_rotate_qk(q, k, rotation.positions[:, start:stop], rotation.frequencies, sections=SECTIONS,
                                   q_weight=rotation.q_weight, k_weight=rotation.k_weight, eps=rotation.eps)
        return q, k, v

    _, plain = run(residency, hidden, project, None)
    _, want = run(residency, hidden, project_and_rotate, None)
    runner, got = run(residency, hidden, project, rotation)
    assert torch.equal(got, want) and not torch.equal(got, plain)

    # Against 64 bits, from the 16-bit projections.
    qkv = (hidden.cuda() @ w).cpu().double().view(TOKENS, HEADS + 2 * KV_HEADS, DIM)
    turn = [rotated(normalized(x, g.cpu(), 1e-5), rotation.positions.cpu(), rotation.frequencies.cpu(), SECTIONS, "halves")[0]
            for x, g in ((qkv[:, :HEADS], rotation.q_weight), (qkv[:, HEADS : HEADS + KV_HEADS], rotation.k_weight))]
    ref = torch.zeros((TOKENS, HEADS, DIM), dtype=torch.float64)
    for first, last in ((0, 40), (40, TOKENS)):
        for h in range(HEADS):
            logits = turn[0][first:last, h] @ turn[1][first:last, h // 2].t() * DIM**-0.5
            mask = torch.ones_like(logits, dtype=torch.bool).tril()
            ref[first:last, h] = torch.softmax(logits.masked_fill(~mask, -torch.inf), -1) @ qkv[first:last, HEADS + KV_HEADS + h // 2]
    assert float((got.double().view_as(ref) - ref).abs().max()) <= 2e-2

    # The producer alone hands out the rotated rows.
    producer = runner.project_qkv_to_device if residency == "hbm" else runner.project_qkv_to_host
    with torch.inference_mode():
        q, k, v = producer(hidden, project, qk_rotation=rotation)
    torch.cuda.synchronize()
    assert float((q.cpu().double() - turn[0]).abs().max()) <= 2**-8 * float(turn[0].abs().max()) * 2
    assert torch.equal(v.cpu().double(), qkv[:, HEADS + KV_HEADS :])


def test_functional_form_and_refusals():
    hidden, weight, rotation = parts()
    w = weight.cuda()

    def project(tile, start, stop):
        return (tile @ w).view(stop - start, HEADS + 2 * KV_HEADS, DIM).split([HEADS, KV_HEADS, KV_HEADS], dim=1)

    _, want = run("host", hidden, project, rotation)
    cu = torch.tensor([0, 40, TOKENS], dtype=torch.int32)
    config = StreamingAttentionConfig(backend="hip", q_chunk_tokens=41, kv_chunk_tokens=29)
    got = streaming_projected_self_attention(
        hidden, cu, q_heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, project_qkv=project,
        output_projector=lambda tile, start, stop: tile, output_features=HEADS * DIM, attention_config=config,
        pipeline_config=ProjectionPipelineConfig(projection_chunk_tokens=31), causal=True, qk_rotation=rotation)
    assert torch.equal(got, want)
    short = QKRotation(positions=rotation.positions[:, :-1], frequencies=rotation.frequencies, sections=SECTIONS)
    with pytest.raises(ValueError, match="whole call"):
        run("hbm", hidden, project, short)
    # A refusal inside the pipeline leaves it usable.
    with pytest.raises(ValueError, match="positions"):
        run("hbm", hidden, project, QKRotation(frequencies=rotation.frequencies))
    assert torch.equal(run("hbm", hidden, project, rotation)[1], want)
