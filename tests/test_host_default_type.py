"""No buffer of the package takes torch's default type: its address goes to kernels that write fp32, past its end
if a program has set a 16-bit default.  Read from the sources, without a device."""

import ast
from pathlib import Path

import boundflow_amd

FACTORIES = {"empty", "zeros", "ones", "full", "eye", "rand", "randn"}


def test_device_buffers_name_their_type():
    nameless = []
    for path in sorted(Path(boundflow_amd.__file__).parent.glob("*.py")):
        for node in ast.walk(ast.parse(path.read_text())):
            if not (isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute)
                    and isinstance(node.func.value, ast.Name) and node.func.value.id == "torch"
                    and node.func.attr in FACTORIES):
                continue
            given = {k.arg for k in node.keywords}
            if "device" in given and "dtype" not in given:
                nameless.append(f"{path.name}:{node.lineno}")
    assert not nameless, nameless
