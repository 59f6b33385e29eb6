"""The active sequences of the Node host's dispatches over sequences, on the CPU."""
from test_node_host import needs_node, run_node


@needs_node
def test_shapes():
    assert "host_cpu_sequences ok" in run_node("host_cpu_sequences.js")
