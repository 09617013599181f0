"""A memory that a model writes, searches exactly and reads: the operators of
``winnex_madhava.memory`` around the engine.

A projection head (layer norm, then a linear layer) turns states into rows of
128; the rows go into a cache of u8 codes, which is also the corpus of the
exact u8 search; queries take the same way, find their nearest rows and attend
over what is stored there; the loss of what they read trains the head's norm
and projection on the query side.

Run on a B200 after the build:  python examples/memory.py
"""
from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "winnex-madhava_b200"))

import torch

import winnex_madhava as wm
from winnex_madhava import memory

STATE, ROW, HEAD, FOUND = 768, 128, 64, 10
LO, STEP = -4.0, 8.0 / 255.0  # the codes' map: rows of about unit variance


def project(states, norm, weight):
    """States -> rows: layer norm, then the projection."""
    return memory.linear(memory.layer_norm(states, *norm), weight)


def run(stored=20_000, queries=64, steps=8, seed=0):
    """Fills a memory, searches it and trains a query head on what is read.
    Returns the losses and the share of queries that find their own state."""
    torch.manual_seed(seed)
    device, kind = "cuda", torch.bfloat16
    states = torch.randn(stored, STATE, device=device, dtype=kind)
    norm = (torch.ones(STATE, device=device), torch.zeros(STATE, device=device))
    weight = (torch.randn(ROW, STATE, device=device) * STATE ** -0.5).to(kind)

    # Write: rows become u8 codes as they are written; the values that go with
    # them are kept in int8 with a scale for each head.
    keys = memory.RowCache.empty(stored, ROW, code="uint8", lo=LO, step=STEP)
    values = memory.RowCache.empty(stored, ROW, group=HEAD)
    slots = torch.arange(stored, device=device)
    with torch.no_grad():
        rows = project(states, norm, weight)
    keys.write(slots, rows)
    values.write(slots, rows)

    # Search: the codes are the corpus.  A query's codes are made the same way.
    engine = wm.build_engine(keys.codes.cpu().numpy(), dim=ROW, k=FOUND, metric="l2", speed=True)
    asked = torch.randint(0, stored, (queries,), device=device)
    query_states = states[asked] + 0.1 * torch.randn(queries, STATE, device=device, dtype=kind)
    probe = memory.RowCache.empty(queries, ROW, code="uint8", lo=LO, step=STEP)
    with torch.no_grad():
        probe.write(torch.arange(queries, device=device), project(query_states, norm, weight))
    found = engine.search_batch(probe.codes.cpu().numpy(), k=FOUND).indices
    ids = torch.tensor(found, dtype=torch.int32, device=device).view(queries, FOUND)
    hit = (ids[:, 0] == asked).float().mean().item()

    # Read: attention over the found rows, nearer ones favoured; train the
    # query side to read back the row that was asked for.
    distance = (keys.read(ids) - probe.read(torch.arange(queries, device=device))[:, None]).square().mean(2)
    head_norm = [t.clone().requires_grad_() for t in norm]
    head = weight.float().clone().requires_grad_()
    nearness = torch.zeros((1, 1), device=device, requires_grad=True)
    target = values.read(asked).view(queries, ROW // HEAD, HEAD)
    optimizer = torch.optim.Adam([*head_norm, head, nearness], lr=3e-3)
    losses = []
    for _ in range(steps):
        q = project(query_states, head_norm, head.to(kind)).view(queries, ROW // HEAD, HEAD)
        out, _ = memory.attend(q, ids, keys, values, cap=30.0, bias=-nearness * distance)
        loss = (out.float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses, hit


if __name__ == "__main__":
    losses, hit = run()
    print(f"nearest row is the one asked for: {hit:.3f} of the queries")
    print("loss of what is read, step by step: " + ", ".join(f"{x:.5f}" for x in losses))
