"""The serving example: a request's logits do not depend on how its tokens were
split over steps nor on what else the steps held."""
import numpy as np
import pytest


@pytest.mark.gpu
def test_serving_example(device):
    from examples.serve import Server

    rng = np.random.default_rng(2)
    text = rng.integers(0, 2048, 90).tolist()
    whole = Server(device).step({3: text})[3].astype(np.float64)
    server = Server(device)
    server.step({0: rng.integers(0, 2048, 40).tolist(), 3: text[:50]})
    server.step({0: [7], 3: text[50:83], 5: [1, 2, 3]})
    for t in text[83:89]:
        server.step({0: [11], 3: [t]})
    server.step({0: [5], 2: [9] * 20}, finished=[5])
    parts = server.step({2: [1], 3: text[89:]}, finished=[0])[3].astype(np.float64)
    # The same values rounded to bf16 (2^-9 each) after sums in another order, through two projections.
    assert np.linalg.norm(parts - whole) <= 2.0 ** -6 * np.linalg.norm(whole)
    held = 256 - int(server.free_count.to_numpy()[0])
    assert held == -(-90 // 16) + -(-21 // 16)


@pytest.mark.gpu
def test_serving_example_main(device, capsys):
    from examples.serve import main

    main(8)
    assert "blocks free" in capsys.readouterr().out
