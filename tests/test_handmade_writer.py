"""The writer of oracle/gen_golden_handmade.py makes the stored streams, and the PCM recorded for them is what it was made from."""
import numpy as np

from oracle import gen_golden_handmade as H


def test_writer_makes_the_stored_streams(handmade_streams):
    made = H.build_streams()
    assert sorted(made) == sorted(handmade_streams)
    for name, (data, pcm) in made.items():
        want, recorded = handmade_streams[name]
        assert data == want, name
        assert np.array_equal(recorded, pcm.astype(np.int32).reshape(recorded.shape)), name
