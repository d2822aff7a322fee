"""Frame attention: the tokens of a target frame look into the visible tokens of many reference frames.

`utils.correlation.compute_masked_4d_correlation` scores every (target, reference) pixel pair, which is why it runs on one pair or on
16 x 16 maps.  These functions answer the same question for whole feature maps and long frame windows: keys are cut into blocks of
64 or 128 consecutive tokens, every group of queries picks the blocks whose mean key fits it best, and attends to the visible keys of
those alone.  Used together:

    pos  = frame_positions(frames, h, w, device)                       # (frames * h * w, 3): time, row, column
    q, k = rotate_positions(q, pos_target, sections), rotate_positions(k, pos, sections)
    means, counts = block_means(k, visible)                            # kept with the keys; new frames add blocks
    blocks = select_blocks(q, means, counts, top_k)
    out  = block_attention(q, k, v, blocks, visible)

Tokens are (batch, token, head, channel) in fp32, bf16 or fp16 (maps (B,C,F,H,W): maps.flatten(2).transpose(1, 2).unflatten(2, (heads, C // heads))), any strides (a view whose rows do not start on 16 bytes is copied);
several query heads may share a key head.  `visible` (batch, token) is a float map as everywhere in this package (seen where
> 0.5; a bool tensor is taken too); holes may hold anything.  HIP kernels of csrc/tcl_rope.hip, tcl_select.hip and tcl_attn.hip through the C
ABI (include/tcl.h)."""
import torch

from .. import _ops


def frame_positions(frames, height, width, device, first_frame=0):
    """Positions (frames * height * width, 3) fp32 of the tokens of a clip, frame after frame and row after row: (time, row, column)."""
    t = torch.arange(first_frame, first_frame + frames, device=device, dtype=torch.float32)
    y = torch.arange(height, device=device, dtype=torch.float32)
    x = torch.arange(width, device=device, dtype=torch.float32)
    return torch.stack(torch.meshgrid(t, y, x, indexing="ij"), dim=-1).reshape(frames * height * width, 3)


def rotate_positions(x, positions, sections, base=10000.0, interleaved=False):
    """Rotary positions over several axes.  x (B,N,H,D), D even up to 256; positions (N,A) or (B,N,A), fp32 or int32; `sections`: the A even
    numbers of channels that belong to each axis, in order (channels behind the last one pass through).  Pair i of a section of d
    channels turns by position * base^(-2i/d): channels (i, i + d/2) of the section, or (2i, 2i + 1) if `interleaved`.
    Angles are formed in 64 bits (far positions keep their phase).  Differentiable in x (a forward-mode tangent is refused).  -> like x."""
    return _ops.rotate_positions(x, positions, sections, base, interleaved)


def block_means(k, visible=None, block=64):
    """Summary of the keys k (B,N,H,D): the mean of the visible keys of each block of `block` (64 or 128) consecutive tokens.
    -> means fp32 (B,H,ceil(N/block),D), counts int32 (B,ceil(N/block)) (visible keys; a block without any has mean 0).
    Data for select_blocks, not differentiable; a cache that grows by whole blocks appends the new blocks' rows."""
    return _ops.block_means(k, visible, block)


def select_blocks(q, means, counts, top_k, q_block=64):
    """Blocks for each group of queries.  q (B,N,H,D); a group is `q_block` consecutive tokens (1: every token chooses for itself) with
    the query heads of one key head.  Block j scores <sum of the group's queries, means[j]>, in 64 bits; the `top_k` best blocks that
    have a visible key are chosen, ties to the lower index (a score of -inf or NaN is not).  Up to 16,384 blocks.  -> int32 (B, key heads, ceil(N/q_block), top_k), ascending, -1 behind the
    last.  Not differentiable."""
    return _ops.select_blocks(q, means, counts, top_k, q_block)


def block_attention(q, k, v, blocks, visible=None, block=64, q_block=64, scale=None, return_lse=False):
    """softmax(scale q k^T) v over the visible keys of the chosen blocks; a query that sees no key gets 0.
    q (B,Nq,Hq,D), k, v (B,Nk,Hkv,D), Hq a multiple of Hkv, D a multiple of 8 up to 128; `blocks` int32 (B,Hkv,ceil(Nq/q_block),top_k) as
    from select_blocks (any order; indices outside the cache are skipped, repeated ones count once; up to 2048 per group); `scale`
    (finite, of any sign) defaults to D^-1/2.  Differentiable (once; a forward-mode tangent is refused) in q, k, v.  -> out (B,Nq,Hq,D) [, lse (B,Hq,Nq) fp32: natural logarithm of the softmax
    denominator, -inf where nothing is seen; not differentiable].
    fp32 inputs run on the fp32 matrix pipe; under autocast q, k, v take the autocast type.
    All sums and statistics are fp32.  16-bit types: the probabilities are rounded to the type before they meet the values, one more rounding than that of the
    result (errors of out together 1.0 to 1.4 times that alone).  So are, in the gradients, probabilities and score gradients where an item's sums are long
    (1.4 to 1.5 times); heads of fewer than 64 channels, groups that can see up to 512 keys and key heads with up to 2,048 query rows take
    both in two parts (1.0 to 1.1 times).  Scores (scale q k) have to stay below 10^9, in fp16 below 2 10^7.
    Few tokens (one, or any number too small to fill the GPU) are served by splitting their keys over workgroups."""
    return _ops.block_attention(q, k, v, blocks, visible, block, q_block, scale, return_lse)
