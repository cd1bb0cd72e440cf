"""The one-launch sort's accesses to the shared memory of other blocks, in the order of its source.

A block's shared memory exists from the block's start to its end, and only a barrier of the cluster tells the others that it
has started.  Whether a launch without that barrier goes wrong depends on the order in which the blocks start, so no run on a
device can be relied on to show it; the source can."""
import os
import re

import llm720_b200

SOURCE = os.path.join(os.path.dirname(llm720_b200.__file__), "csrc", "row_sort.cu")


def _body(name):
    """The braces behind the kernel's name, without comments."""
    text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    at = text.index("{", text.index(name + "("))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(name)


def test_no_block_is_written_to_before_the_whole_cluster_has_started():
    body = _body("sort_cluster_kernel")
    calls = re.findall(r"\b(cluster_started_arrive|cluster_started_wait|cluster_sync|store_remote|remote)\s*\(", body)
    remote = min(calls.index("store_remote"), calls.index("remote"))
    # some barrier of the cluster lies in front of the first access ...
    assert "cluster_sync" in calls[:remote] or "cluster_started_wait" in calls[:remote], calls
    # ... and a split one is entered by every thread, at the kernel's first statement, and waited for in the first pass
    if "cluster_started_wait" in calls[:remote]:
        assert calls[0] == "cluster_started_arrive" and calls.count("cluster_started_arrive") == 1
        assert re.match(r"\{\s*cluster_started_arrive\(\);", body)
        assert re.search(r"if \(p == 0\) cluster_started_wait\(\);", body) and calls.count("cluster_started_wait") == 1


def test_no_block_leaves_while_others_may_write_to_it():
    """In the last pass the results go to global memory, and the one exchange before them ends with a barrier."""
    body = _body("sort_cluster_kernel")
    last = body.index("if (last) break;")
    assert "store_remote" not in body[last:]
    assert re.search(r"if \(last\) \{\s*if \(to < n\)", body[:last])
    assert body[:last].rindex("cluster_sync();") > body[:last].index("store_remote")
