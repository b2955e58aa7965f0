"""page_slots refuses what its 32-bit arithmetic does not hold."""
from miori_b200._lib import lib

OK = 0x1000  # aligned, never dereferenced: validation fails first


def test_pages_and_tables_that_are_too_large():
    def slots(requests=4, width=3, page=16):
        return lib.miori_page_slots(OK, OK, OK, OK, OK, OK, OK, OK + 128, OK + 64, OK + 256, requests, width, page, 5, 4, 0, None)

    for call, text in ((lambda: slots(page=2 ** 30 + 1), b"2^30"), (lambda: slots(page=2 ** 32 - 16), b"2^30"), (lambda: slots(width=2 ** 31), b"2^31"),
                       (lambda: slots(requests=16384, width=2 ** 17), b"2^31"), (lambda: slots(requests=1, width=2 ** 32 - 1), b"2^31")):
        assert call() == -1
        assert text in lib.miori_last_error(), lib.miori_last_error()
