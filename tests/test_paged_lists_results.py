"""Results of the page lists' native entry that overlap what it reads."""

from __future__ import annotations

import pytest

from autosage_amd import _native


def test_results_over_lengths_or_changes_are_refused():
    """One workgroup would give the right results, several would read what others have written."""
    path = _native.package_library_path()
    if not path.exists():
        pytest.skip("HIP library not built")
    lib = _native.open_library(path)
    at = {name: 4096 * (i + 1) for i, name in enumerate(("table", "lengths", "change", "free", "count", "new", "ptr",
                                                           "positions", "slots", "ws"))}

    def resize(sequences=3, tokens=5, **over):
        p = {**at, **over}
        return lib.as_paged_cache_resize(p["table"], 4, 4, p["lengths"], p["change"], p["free"], 9, p["count"], 4, p["new"],
                                         p["ptr"], p["positions"], p["slots"], sequences, tokens, p["ws"], 1 << 20, None)

    for name, count in (("new", 3), ("ptr", 4), ("positions", 5), ("slots", 5)):
        for read in ("lengths", "change"):
            for place in (at[read], at[read] + 16, at[read] - 8 * (count - 1)):
                assert resize(**{name: place}) == 1
                assert lib.as_last_error().startswith(b"the results must lie apart")
