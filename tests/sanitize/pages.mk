# The host code of the operators around a paged cache under AddressSanitizer and
# UndefinedBehaviorSanitizer, linked into kvq_pages_check (as Makefile does for
# kvq_host_check; the device code is built but never launched).
include $(dir $(abspath $(lastword $(MAKEFILE_LIST))))Makefile
.DEFAULT_GOAL := pages
PAGES := $(foreach n,kvq_pages kvq_select kvq_pages_capi,$(BUILD)/$(n).o)

pages: $(BUILD)/kvq_pages_check

$(BUILD)/kvq_pages_capi.o: $(CSRC)/kvq_pages_capi.cpp $(DEPS)
	@mkdir -p $(BUILD)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(BUILD)/kvq_pages_check.o: $(HERE)kvq_pages_check.cpp $(DEPS)
	@mkdir -p $(BUILD)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(BUILD)/kvq_pages_check: $(OBJS) $(PAGES) $(BUILD)/kvq_pages_check.o
	$(HIPCC) --offload-arch=gfx950 $(SAN) -o $@.tmp $^ && mv $@.tmp $@

.PHONY: pages
