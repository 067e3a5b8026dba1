"""What the kernels' sources and the wrappers have to say alike, read from the sources (no GPU)."""
import os
import re

import tgo_b200

CSRC = os.path.join(os.path.dirname(tgo_b200.__file__), "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def kernel(name, file):
    text = source(file)
    start = text.index(f" {name}(")
    return re.sub(r"//.*", "", text[start:text.index("\n}\n", start)])


def test_a_wait_that_ran_out_in_one_thread_is_known_to_all():
    """The copying kernel of constrained logits: one thread settles the copies under way when the block gives up, whichever
    thread's wait ran out, so each has to have the block's answer and not its own."""
    body = kernel("constrain_stream_kernel", "drafts.cu")
    wait = body.index("tg_wait(&full[b]")
    leave = body.index("break;", wait)
    assert re.search(r"\bok = __syncthreads_and\(ok\);\s*if \(!ok\) $", body[wait:leave])
    assert re.search(r"if \(!ok\) tg_settle_copies\(full", body[leave:])
    # nobody's own answer between the two
    assert "__syncthreads_or(!ok)" not in "".join(source(f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def test_limits_are_those_of_the_sources():
    from tgo_b200.kernels import ops
    tree, drafts = source("attention_tree.cu"), source("drafts.cu")
    assert [int(re.search(rf"#define {name} (\d+)", text).group(1)) for name, text in (("TREE_NODES", tree), ("DR_NODES", drafts))] == \
        [ops.TREE_NODES] * 2
    assert f"dh > {ops.TREE_HEAD} " in tree[tree.index("TGO_API int tgo_attention_tree(const"):]
    assert int(re.search(r"#define LC_ROWS (\d+)", drafts).group(1)) == 65535
