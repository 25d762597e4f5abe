from . import embedding, grid_sample, group_norm, grouped_linear, spconv, utils  # noqa: F401
