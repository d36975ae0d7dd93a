from greyhound_b200.nn import functional, utils

__all__ = ["functional", "utils"]
