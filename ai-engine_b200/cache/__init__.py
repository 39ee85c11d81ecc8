from .manager import CacheGroup, PagedCache, group_requests, host
from .tables import StepTables, step_tables

__all__ = ["CacheGroup", "PagedCache", "StepTables", "group_requests", "host", "step_tables"]
