"""The library that the golden vectors were recorded from is not run here: prebuilt machine code that ships inside the reference
is neither loaded nor executed.  What it wrote and reported stands in ``tests/golden/``; nothing outside those vectors is
pinned to it.  ``tests/test_oracle_vs_reference.py`` asks ``available()`` and is skipped as a whole.
"""


def available():
    return False
