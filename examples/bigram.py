"""A byte-level bigram language model: the vocabulary operators as a program uses them.

The model is one table: row t holds the logits of the byte that follows byte t,
so a step needs no matrix product. Training: ``F.embedding`` looks the rows up,
``F.cross_entropy`` gives the loss, ``ft.grad`` goes back through both to the
table, and one ``ft.evaluate`` runs it all with the update. Generation: the
rows of the last bytes, ``F.adjust_logits`` with each sequence's own history
and the bytes that may be chosen, Gumbel noise and ``ft.argmax``.

    python examples/bigram.py [FILE]        (default: this file)
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import fugatensor_b200 as ft
import fugatensor_b200.nn.functional as F

VOCAB = 256


def train(text: bytes, steps=200, batch=8192, rate=200.0, seed=0):
    """The table after `steps` of gradient descent on random positions of `text`, and each step's loss."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    data = torch.frombuffer(bytearray(text), dtype=torch.uint8).to("cuda", torch.int32)
    table = ft.tensor(torch.zeros(VOCAB, VOCAB, device="cuda"))
    losses = []
    for _ in range(steps):
        at = torch.randint(0, len(text) - 1, (batch,), device="cuda", generator=g)
        ids, targets = ft.tensor(data[at], dtype=ft.int32), ft.tensor(data[at + 1], dtype=ft.int32)
        loss = F.cross_entropy(F.embedding(table, ids), targets, z_loss=1e-4)
        updated = table - ft.grad(loss, table) * rate
        ft.evaluate(loss, updated)
        table = updated
        losses.append(loss)
    return table, [v.item() for v in losses]


def allow(tokens):
    """The bit mask [VOCAB / 32] of a set of tokens."""
    words = [0] * (VOCAB // 32)
    for t in tokens:
        words[t // 32] |= 1 << t % 32
    return torch.tensor([w - (w >> 31 << 32) for w in words], dtype=torch.int32, device="cuda")


def generate(table, prompt: bytes, sequences=4, length=80, seed=0, repetition=1.05, frequency=0.02, allowed=range(32, 127)):
    """`sequences` continuations of `prompt` by `length` bytes each, out of the `allowed` ones."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.full((sequences, len(prompt) + length), -1, dtype=torch.int32, device="cuda")
    tokens[:, :len(prompt)] = torch.tensor(list(prompt), dtype=torch.int32)
    prompts = ft.tensor(torch.full((sequences,), len(prompt), device="cuda"), dtype=ft.int32)
    mask = ft.tensor(allow(allowed).expand(sequences, -1), dtype=ft.int32)
    for n in range(len(prompt), len(prompt) + length):
        logits = F.embedding(table, ft.tensor(tokens[:, n - 1], dtype=ft.int32))
        logits = F.adjust_logits(logits, ft.tensor(tokens, dtype=ft.int32), ft.tensor(torch.full((sequences,), n, device="cuda"), dtype=ft.int32),
                                 prompt_lengths=prompts, repetition=repetition, frequency=frequency, allowed=mask)
        noise = -torch.log(-torch.log(torch.rand(sequences, VOCAB, device="cuda", generator=g)))
        tokens[:, n] = ft.evaluate(ft.argmax(logits + ft.tensor(noise), axis=1)).torch()
    return [bytes(row) for row in tokens[:, len(prompt):].tolist()]


if __name__ == "__main__":
    source = Path(sys.argv[1] if len(sys.argv) > 1 else __file__).read_bytes()
    model, history = train(source)
    print(f"loss {history[0]:.3f} -> {history[-1]:.3f} nats per byte")
    for line in generate(model, b"def "):
        print("def " + line.decode())
