"""The shape of a tree of drafted tokens (speculative decoding).

A tree is its parents' list: node 0 is the root (the last token already
decided, not yet in the cache), node i's parent is an earlier node.  Node i
of a sequence with ``ctx`` cached tokens takes slot ``ctx + i`` and position
``ctx + depth(i)``.  A node attends to the cache, to its ancestors and to
itself; ``mask`` packs that as the int32 words ``paged_tree_attention``
reads.  No counterpart in the reference, which decodes one token per pass.
"""

from __future__ import annotations

import numpy as np


class DraftTree:
    """Parents, depths and attention mask of one tree topology."""

    def __init__(self, parents) -> None:
        par = np.asarray(parents, dtype=np.int64)
        if par.ndim != 1 or len(par) == 0:
            raise ValueError("a draft tree has at least its root")
        if (par[1:] < 0).any() or (par[1:] >= np.arange(1, len(par))).any():
            raise ValueError("every node but the root needs an earlier node as its parent")
        self.parents = par.astype(np.int32)
        self.parents[0] = -1
        self.depths = np.zeros(len(par), dtype=np.int32)
        seen = np.eye(len(par), dtype=bool)
        for i in range(1, len(par)):
            self.depths[i] = self.depths[par[i]] + 1
            seen[i] |= seen[par[i]]
        self._seen = seen

    @classmethod
    def from_widths(cls, widths) -> "DraftTree":
        """A full tree: every node of level d has ``widths[d]`` children."""
        parents, level = [-1], [0]
        for w in widths:
            if w < 1:
                raise ValueError("a level needs at least one child per node")
            nxt = []
            for node in level:
                for _ in range(w):
                    nxt.append(len(parents))
                    parents.append(node)
            level = nxt
        return cls(parents)

    def __len__(self) -> int:
        return len(self.parents)

    @property
    def max_depth(self) -> int:
        return int(self.depths.max())

    def level(self, depth: int) -> np.ndarray:
        """The nodes at ``depth``, in order."""
        return np.nonzero(self.depths == depth)[0]

    def mask(self, words: int | None = None) -> np.ndarray:
        """int32 (nodes, words): bit j % 32 of word j // 32 of row i says that i sees j."""
        n = len(self)
        need = (n + 31) // 32
        words = need if words is None else int(words)
        if words < need:
            raise ValueError(f"{n} nodes need {need} mask words")
        bits = np.zeros((n, words * 32), dtype=np.uint8)
        bits[:, :n] = self._seen
        packed = np.packbits(bits, axis=1, bitorder="little")
        return np.ascontiguousarray(packed).view("<i4").astype(np.int32).reshape(n, words)
