"""The example that trains in the clear and answers under encryption: the loss
falls, and the encrypted block's output is the cleartext operators'."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_trained_in_the_clear_answered_under_encryption():
    import next_item
    model, successor, losses = next_item.train(steps=150, batch=512, log=lambda line: print("[next item]", line, flush=True))
    assert losses[-1] < 0.7 * losses[0]
    server = next_item.EncryptedModel(model)
    try:
        for item in (0, 101, 255):
            z = server.ask(item)
            clear = next_item.block(model, model["table"][item:item + 1])[0].cpu().double().numpy()
            print("[next item]", item, np.abs(z - clear).max(), flush=True)
            # encoding at scale 2^50 and float32 weights: 2^-20 of the largest value, as the lookup is held to
            assert np.abs(z - clear).max() <= 2.0 ** -20 * max(1.0, np.abs(clear).max()) * 16
    finally:
        server.close()
