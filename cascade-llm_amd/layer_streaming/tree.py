"""Drafted trees: what the host says of their shape.

The reference decodes one token at a time (tools/run_llama31.py:105-121).  A
step may score several drafted tokens of a sequence instead, a tree of up to
64 nodes whose node 0 is the token drawn last.  ``PagedKVCache.attend_tree``
and ``PagedKVCache.accept`` read the shape as device tensors.
"""

import operator

__all__ = ["tree_masks"]


def tree_masks(parents):
    """(masks, depths) of one tree's nodes, two lists of integers.

    ``parents[i]`` is the place of node i's parent in the tree, before i; node
    0's is -1.  Bit j of ``masks[i]`` says that node i reads node j: itself and
    its ancestors (an int64: node 63's bit is the sign).  A node of depth d
    continues the text at position past + d."""

    parents = [operator.index(parent) for parent in parents]
    if len(parents) > 64:
        raise ValueError("a tree has at most 64 nodes, this one {}".format(len(parents)))
    masks, depths = [], []
    for node, parent in enumerate(parents):
        if node == 0:
            if parent != -1:
                raise ValueError("the parent of node 0 is -1")
            masks.append(1)
            depths.append(0)
            continue
        if not 0 <= parent < node:
            raise ValueError("the parent of node {} is {}, not a node before it".format(
                node, parent))
        masks.append(masks[parent] | 1 << node)
        depths.append(depths[parent] + 1)
    return [mask - (1 << 64) if mask >> 63 else mask for mask in masks], depths
