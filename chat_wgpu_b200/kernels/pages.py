"""Block tables, slots and positions of a step over a paged cache (no reference
counterpart: its cache is one contiguous row per position)."""
from .. import _lib
from ..context import Buffer
from ._util import Prepared


class PagePlan(Prepared):
    """Pages, slots and positions of a step's tokens from the request lengths
    (cw_page_plan).  Every buffer holds i32; `table` is updated in place.  `used`
    above n_free means that pages ran out: the tokens without one have slot -1."""

    _fn = "cw_page_plan"
    _struct = _lib.PagePlanArgs

    def __init__(self, ctx, lens: Buffer, news: Buffer, free_pages: Buffer | None, table: Buffer,
                 starts: Buffer, positions: Buffer, slots: Buffer, owners: Buffer, used: Buffer,
                 n_req: int, page_size: int, max_pages: int, n_free: int, max_tokens: int,
                 depths: Buffer | None = None):
        super().__init__(
            ctx, lens=lens, news=news, free_pages=free_pages, table=table, depths=depths,
            starts=starts, positions=positions, slots=slots, owners=owners, used=used,
            n_req=n_req, page_size=page_size, max_pages=max_pages, n_free=n_free,
            max_tokens=max_tokens)
