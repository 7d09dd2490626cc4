"""Parameters of the programs around the training operators, looked at when a program is built: no device is needed."""
import numpy as np
import pytest

import tensorfrost_amd.host as tf


@pytest.fixture(scope="module")
def codegen():
    tf.initialize(tf.codegen)
    yield tf
    tf.shutdown()


def bits(x):
    return int(np.float32(x).view(np.int32))


ALLOWED = {"layer_norm": [bits(1e-3)], "layer_norm_backward": [], "embedding": [bits(-2.0)], "embedding_backward": [57, bits(3.0)],
           "newton_schulz": [3, bits(1e-6), bits(1.5), bits(-0.5), bits(0.0)], "embed_norm_dense": [bits(1e-5), bits(2.0)]}


@pytest.mark.parametrize("name", ALLOWED)
def test_parameters_beyond_those_of_a_program_are_refused(codegen, name):
    """Coefficients for every step, say, which the program would have read as those of one."""
    params = ALLOWED[name]
    tf.compile(name, params)
    with pytest.raises(tf.TFHostError, match=f"{name} takes at most {len(params)} parameters"):
        tf.compile(name, params + [bits(1.0)])


@pytest.mark.parametrize("name", [n for n in ALLOWED if ALLOWED[n]])
def test_parameters_are_words_of_32_bits(codegen, name):
    tf.compile(name, [0x7FFFFFFF] + ALLOWED[name][1:])
    tf.compile(name, ALLOWED[name][:-1] + [0xBF800000])  # the bits of a negative number, unsigned
    for bad in ((1 << 32) + 5, -(1 << 31) - 1):
        with pytest.raises(tf.TFHostError, match="does not fit 32 bits"):
            tf.compile(name, [bad] + ALLOWED[name][1:])
