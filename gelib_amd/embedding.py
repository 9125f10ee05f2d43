"""Rows of a table by tokens, the first layer of a network over points: what each of them is (the element of an atom, the type of a
cell).  The lookup's counterpart in the reference is a gather of slices (python/src/gelib/gather_map.py); the gradient's is its inverse."""
from gelib_amd.gelib_common import backend


def embedding(tokens, table, scale=1.0):
    """scale * table[tokens]: (*tokens.shape, channels) from int32 or int64 tokens of any shape and a table (rows, channels) of float32,
    bfloat16 or float16 values on the GPU.

    A token below zero (padding) gives a row of zeros and no gradient; one that is `rows` or more gives a row of NaN and no gradient: tokens
    are read on the GPU only.  Differentiable in the table: its gradient is dense, summed in float32 in an order that does not change
    from run to run, and rounded once; twice by torch's own operations, which forward-mode derivatives, function transforms,
    tracing and dispatch modes get from the start."""
    return backend().embedding(tokens, table, float(scale))
