"""CPU test: a chain whose recording fails keeps no handle of the graph that it
had destroyed before."""
import pytest

from atlas_amd.chains import GemmaPrefillChunk, LlamaDecodeStep, SharedPromptDecode
from atlas_amd.decode import GemmaDecodeStep


class Runtime:
    def __init__(self):
        self.live, self.next, self.fails = set(), 1, False

    def graph_begin(self):
        pass

    def graph_end(self):
        self.next += 1
        self.live.add(self.next)
        return self.next

    def graph_destroy(self, graph):
        self.live.remove(graph)  # KeyError: destroyed twice


@pytest.mark.parametrize("kind", [LlamaDecodeStep, GemmaPrefillChunk, SharedPromptDecode, GemmaDecodeStep])
def test_a_failed_recording_leaves_no_graph_behind(kind):
    chain = object.__new__(kind)
    chain.rt, chain.graph = Runtime(), None
    chain.enqueue = lambda: None
    first = chain.capture()
    assert chain.graph == first and chain.rt.live == {first}

    def fails():
        raise ValueError("no")

    chain.enqueue = fails
    with pytest.raises(ValueError, match="no"):
        chain.capture()
    assert chain.graph is None and not chain.rt.live
    chain.enqueue = lambda: None
    chain.capture()
    chain.close()
    assert chain.graph is None and not chain.rt.live
