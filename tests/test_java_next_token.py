"""CPU checks of the Java adapter's next-token binding (as test_java_binding.py:
the descriptor, the typed wrapper and the call against the C header)."""
import re

from tests.test_java_binding import CARRIER, header_functions, java_descriptors, java_text


def test_next_token_descriptor_and_wrapper_match_the_header():
    ret, params, critical = java_descriptors()["gollek_hip_next_token"]
    assert (ret, params) == header_functions()["gollek_hip_next_token"]
    assert critical  # float[] and int[] go in as heap segments
    m = re.search(r"\n\s+int nextToken\(([^)]*)\)\s*\{(.*?)\n        \}", java_text(), flags=re.S)
    decl = [p.strip().rsplit(" ", 1) for p in m.group(1).split(",")]
    assert [t for t, _ in decl] == [CARRIER[p] for p in params]
    call = re.search(r"return \(int\) nextToken\.invokeExact\(([^)]*)\)", m.group(2))
    assert [a.strip() for a in call.group(1).split(",")] == [n for _, n in decl]


def test_try_next_token_passes_its_arguments_in_order():
    body = re.search(r"static boolean tryNextToken\(.*?\n    \}\n", java_text(), flags=re.S).group(0)
    call = re.search(r"b\.nextToken\((.*?)\);\n", body, flags=re.S).group(1)
    args = [a.strip() for a in re.split(r",(?![^()]*\))", " ".join(call.split()))]
    assert args == ["w", "MemorySegment.ofArray(vector)", "(long) vector.length", "temperature", "topK", "topP", "minP",
                    "u", "MemorySegment.ofArray(token)", "MemorySegment.NULL", "MemorySegment.NULL", "err",
                    "(long) ERR_LEN"]
    assert "token.length < 1" in body


def test_a_library_without_the_entry_serves_the_others():
    # ABI 1.0 has no gollek_hip_next_token: its handle is optional, the others' are not
    text = java_text()
    optional = re.findall(r'lookup\.find\("(\w+)"\)\.isEmpty\(\) \? null\s*: downcall\(linker, lookup, "(\w+)"', text)
    assert optional == [("gollek_hip_next_token", "gollek_hip_next_token")]
    body = re.search(r"static boolean tryNextToken\(.*?\n    \}\n", text, flags=re.S).group(0)
    assert "if (b == null || !b.hasNextToken() || !supportsType(tensor.typeId())) {\n            return false;" in body
    assert body.index("hasNextToken") < body.index("handle(b, ")
    assert re.search(r"boolean hasNextToken\(\) \{\s*return nextToken != null;", text)
