"""Attention over the points of a document (the atoms of a molecule, the cells of a grid): invariant channels of every point from those of
all others, nearer ones more than far ones.  No counterpart in the reference, whose layers meet neighbours through gather."""
from gelib_amd.gelib_common import backend


def attention(q, k, v, points=None, slopes=None, key_points=None, lengths=None, query_lengths=None, starts=None, query_starts=None, scale=None):
    """y_i = sum_j softmax_j(scale q_i . k_j - slopes[h] |points_i - key_points_j|) v_j over the keys j of i's document, zero where there
    are none; float32, bfloat16 or float16 tensors of one type on the GPU.

    q (samples, n_q, heads, dim), k and v (samples, n_k, kv_heads, dim): a document is a sample, of which the first lengths[n] keys and
    query_lengths[n] queries exist (int32; None: all).  What does not exist is not read, and is zero in the result and in gradients.
    q (rows, heads, dim), k and v (rows, kv_heads, dim): documents lie one behind the other, document d the keys starts[d] to
    starts[d + 1] and the queries query_starts[d] to query_starts[d + 1] (int32, ascending, one more than documents; query_starts None: the
    same rows).  Rows in no document are zero.  Lengths and starts are read on the GPU only, and held to the rows there are.

    Heads h of q stand on heads h / (heads / kv_heads) of k and v.  dim is at most 128; a head's channels are contiguous, other strides
    as they come.  points and key_points (rows of q and of k, three coordinates each; key_points None: points) and slopes (heads) are float32.
    Points are finite numbers below 1e38; a distance above 1.8e19, whose square float32 does not hold, counts as that.  scale None: dim ** -0.5.
    One query a sample (n_q = 1) reads a sample out.

    Scores, softmax and sums are float32; 16-bit types round its values to their own for the second product, and results once, so that errors are
    those of rounding the result times 1.4.  Differentiable
    in q, k, v, points, slopes and key_points (points in one place have no direction and add nothing to each other's gradient), twice by torch's
    own operations, which forward-mode derivatives, function transforms, tracing and dispatch modes get from the start.  Those form the
    scores of all rows with all rows of packed documents, and what is no number in one document reaches the others there.  float16
    gradients are float16 values: losses are scaled up as usual with that type (what leads to them is kept in range, whatever their size)."""
    return backend().attention(q, k, v, points, slopes, key_points, lengths, query_lengths, starts, query_starts, scale)
