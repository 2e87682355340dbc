"""The FFM descriptors of the integration guide against the header's prototypes, argument by argument (no GPU)."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def prototypes():
    """name -> [return layout, argument layouts ...] of every function the header declares."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gollek_kernels.h")).read(), flags=re.S)
    text = re.sub(r"^\s*#[^\n]*", "", text, flags=re.M)
    kinds = {"int": "JAVA_INT", "unsigned": "JAVA_INT", "float": "JAVA_FLOAT", "size_t": "JAVA_LONG"}

    def layout(decl):
        decl = decl.strip()
        return "ADDRESS" if "*" in decl else "JAVA_LONG" if "long long" in decl else kinds[decl.replace("const ", "").split()[0]]

    return {m[1]: [layout(m[0] + " f")] + [layout(a) for a in m[2].split(",") if a.strip() not in ("", "void")]
            for m in re.findall(r"GOLLEK_API\s+([\w\s]+?\*?)\s*(\w+)\s*\(([^)]*)\)", text)}


def descriptors():
    """name -> layouts of every downcall handle that the guide shows."""
    for f in sorted(os.listdir(ROOT)):
        if f.endswith(".md"):
            text = open(os.path.join(ROOT, f)).read()
            code = "\n".join(re.findall(r"```java\n(.*?)```", text, flags=re.S))
            if "downcallHandle" in code:
                code = re.sub(r"//[^\n]*", "", code)
                return {m[0]: [a.strip() for a in m[1].split(",") if a.strip()] for m in re.findall(
                    r'find\("(\w+)"\)[^;]*?FunctionDescriptor\.of\(([^)]*)\)', code, flags=re.S)}
    return {}


SHOWN = descriptors()


def test_the_guide_shows_the_attention_and_cache_entry_points():
    assert {"gollek_paged_attention_v2", "gollek_paged_attention_prefill", "gollek_paged_attention_varlen",
            "gollek_paged_attention_varlen_workspace_size", "gollek_paged_attention_shared_prefix",
            "gollek_paged_attention_shared_prefix_workspace_size", "gollek_kv_append", "gollek_kv_gather",
            "gollek_kv_migrate"} <= set(SHOWN)


@pytest.mark.parametrize("name", sorted(SHOWN))
def test_descriptor_matches_the_header(name):
    assert SHOWN[name] == prototypes()[name]
