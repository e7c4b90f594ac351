"""Kernels whose blocks reach into each other's shared memory, held to what makes that sound at their start, by reading the sources: a
block of the cluster may not have started yet, and its shared memory may be reached only behind a barrier of the cluster."""
import re

from test_dependent_launches import closing, sources

REMOTE = r"\b(?:ld_cluster\w*|st_cluster\w*|mbar_arrive_cluster)\("
BARRIER = re.compile(r"\b(?:cluster_wait|cluster_sync)\(\)")


def without_local_functions(body):
    """The body without its local functions that reach into other blocks, and what a call of one looks like"""
    names = []
    while True:
        reach = re.compile("|".join([REMOTE] + [rf"\b{n}\(" for n in names]))
        for m in re.finditer(r"auto (\w+) = \[&\]\(", body):
            start = body.index("{", closing(body, m.end() - 1, "()"))
            end = closing(body, start, "{}")
            if reach.search(body[start:end]):
                names.append(m.group(1))
                body = body[:m.start()] + body[end:]
                break
        else:
            return body, reach


def test_a_cluster_has_started_before_it_is_reached_into():
    seen = set()
    for name, text, found in sources():
        for kernel, _, body, _, _ in found:
            body, reach = without_local_functions(body)
            first = reach.search(body)
            if first is None:
                continue
            seen.add(kernel)
            barrier = BARRIER.search(body)
            assert barrier and barrier.start() < first.start(), (name, kernel, first.group())
    assert {"sample_rows_kernel"} < seen and len(seen) >= 5, seen
