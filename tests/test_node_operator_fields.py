"""Fields of the block norm, the 4-bit product and the token scores in the Node
host: a value that is none of the field's is refused, never taken for absent."""
from test_node_host import needs_node, run_node


@needs_node
def test_values_of_no_field_are_refused():
    assert "host_cpu_operator_fields ok" in run_node("host_cpu_operator_fields.js")
