"""A next-item model, trained in the clear and answered under encryption.

    python examples/next_item.py

The model holds a table of items.  An item's row is normalised, goes through a
gated feed-forward block with a cubic activation, and the result is scored
against the same table:

    z = block(layer_norm(table[item]));  p(next) = softmax(<z, table>)

Training takes `helrm_amd.cleartext`: embedding, layer_norm, gated_mlp and
cross_entropy on the GPU.  The trained model is then evaluated on an encrypted one-hot
selector with what the backend has: the normalisation folds into the table
(the norm of a looked-up row is a look-up in the table of normalised rows), so
the encrypted path is a lookup, two Linears, the activation, a product of
ciphertexts and a Linear.  The client decrypts z and scores it in the clear.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from helrm_amd import cleartext as ct  # noqa: E402
from helrm_amd import orion_host as oh  # noqa: E402
from helrm_amd.backend import HipLibrary  # noqa: E402
from helrm_amd.workloads import ACTIVATION3  # noqa: E402

ITEMS, WIDTH, HIDDEN = 256, 16, 32
CUBIC = tuple(reversed(ACTIVATION3))      # lowest degree first


def score(model, z, target, ignore_index=-100):
    return ct.cross_entropy(z, model["table"], target, ignore_index)


def block(model, rows):
    n = ct.layer_norm(rows, model["weight"], model["bias"])
    return ct.gated_mlp(n, model["gate"], model["up"], model["down"], CUBIC)


def train(steps=400, batch=1024, seed=0, log=print):
    """A model of the synthetic sequence item -> next[item]; a tenth of the positions has no target."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).requires_grad_()

    model = {"table": normal(ITEMS, WIDTH, std=0.5),
             "weight": torch.ones(WIDTH, device="cuda", requires_grad=True),
             "bias": torch.zeros(WIDTH, device="cuda", requires_grad=True),
             "gate": normal(HIDDEN, WIDTH, std=WIDTH ** -0.5),
             "up": normal(HIDDEN, WIDTH, std=WIDTH ** -0.5),
             "down": normal(WIDTH, HIDDEN, std=HIDDEN ** -0.5)}
    successor = torch.randperm(ITEMS, generator=gen, device="cuda")
    opt = torch.optim.Adam(model.values(), lr=1e-2)
    losses = []
    for step in range(steps):
        item = torch.randint(ITEMS, (batch,), generator=gen, device="cuda")
        target = successor[item]
        target = torch.where(torch.rand(batch, generator=gen, device="cuda") < 0.1, torch.full_like(target, -100), target)
        loss = score(model, block(model, ct.embedding(item, model["table"])), target)
        opt.zero_grad()
        loss.backward()
        opt.step()
        if step % 50 == 0 or step == steps - 1:
            losses.append(loss.item())
            log(f"step {step}: loss {losses[-1]:.4f}")
    return {k: v.detach() for k, v in model.items()}, successor, losses


class EncryptedModel:
    """The trained model behind the CKKS backend: N = 2^13, nine 50-bit levels."""

    def __init__(self, model, seed=5):
        self.lib = HipLibrary()
        p = oh.Params(13, [60] + [50] * 8, [61] * 3, 50, 192, seed=seed)
        self.scheme = oh.Scheme(p, self.lib)
        rows = ct.layer_norm(model["table"], model["weight"], model["bias"]).cpu().numpy()
        weights = {k: model[k].cpu().numpy() for k in ("gate", "up", "down")}
        self.lookup = oh.LinearLayer(self.scheme, rows.T, level=8, name="lookup").compile()
        self.gate = oh.LinearLayer(self.scheme, weights["gate"], level=7, name="gate").compile()
        self.up = oh.LinearLayer(self.scheme, weights["up"], level=7, name="up").compile()
        self.activation = oh.Activation(self.scheme, ACTIVATION3).compile()
        # the product is taken at level 4: at a scale of that modulus the activation leaves the default scale there
        self.activation.output_scale = self.scheme.moduli()[4]
        self.down = oh.LinearLayer(self.scheme, weights["down"], level=3, name="down").compile()

    def ask(self, item):
        """z of one encrypted item, decrypted."""
        selector = np.zeros(ITEMS, dtype=np.float32)
        selector[item] = 1.0
        x = self.lookup.forward(self.scheme.encrypt(self.scheme.encode(selector, 8)))
        a, u = self.activation.forward(self.gate.forward(x)), self.up.forward(x)
        h = self.lib.MulRelinCiphertextNew(a.ids[0], u.ids[0])
        self.lib.Rescale(h)
        y = self.down.forward(oh.CipherTensor(self.scheme, [h], HIDDEN))
        return self.scheme.decode(self.scheme.decrypt(y))[:WIDTH]

    def close(self):
        self.lib.DeleteScheme()


def main():
    args = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    args.add_argument("--steps", type=int, default=400)
    args.add_argument("--ask", type=int, default=4, help="items to ask for under encryption")
    args = args.parse_args()
    model, successor, _ = train(args.steps)
    server = EncryptedModel(model)
    try:
        for item in range(args.ask):
            z = server.ask(item)
            clear = block(model, model["table"][item:item + 1])[0].cpu().double().numpy()
            scores = model["table"].cpu().double().numpy() @ z
            print(f"item {item}: answer {int(scores.argmax())}, next {int(successor[item])}, "
                  f"largest difference to the clear {np.abs(z - clear).max():.2e}", flush=True)
    finally:
        server.close()


if __name__ == "__main__":
    main()
